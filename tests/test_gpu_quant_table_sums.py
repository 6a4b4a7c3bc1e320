"""Request lengths whose new tokens are more than 32 bits hold together."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from fa_mi355x import capi
from tests.test_quant_host import TABLE

DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
MOST = 2 ** 31 - 1


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [2, 3, 5, 4096, 4097, 9000])
@pytest.mark.parametrize("short", [0, 1, 40])
def test_new_tokens_past_32_bits(batch, short):
    """The first `short` requests grow by 5 tokens, all others to the largest length; each has 4 pages of 16 at most."""
    print(f"case table sums {batch} {short}", flush=True)
    short = min(short, batch - 1)
    before = torch.randint(0, 3, (batch,), generator=torch.Generator().manual_seed(111))
    after = torch.full((batch,), MOST)
    after[:short] = before[:short] + 5
    need = [(int(a) + 15) // 16 if i < short else 4 for i, a in enumerate(after)]
    have = [1 if b else 0 for b in before.tolist()]
    take = sum(n - h for n, h in zip(need, have))
    table = torch.full((batch, 4), -1, dtype=torch.int32)
    table[:, 0] = torch.where(before > 0, torch.arange(batch) + 10 * batch, -1).int()
    free = torch.arange(take, dtype=torch.int32)
    total = 300
    got = table.to(DEV)
    slots, cu, left = fa.update_page_table(got, before.to(**I32), after.to(**I32), free.to(DEV), torch.tensor([take], **I32), 16, total)
    want, top = table.clone(), take
    for b in range(batch):
        for j in range(have[b], need[b]):
            top -= 1
            want[b, j] = top
    assert torch.equal(got.cpu(), want) and left.item() == 0
    new = (after - before).cumsum(0).clamp(max=MOST)
    assert cu.tolist() == [0] + new.tolist()
    want_slots = []
    for b in range(batch):
        for at in range(int(before[b]), min(int(after[b]), total + 3)):
            want_slots.append(int(want[b, at // 16]) * 16 + at % 16 if at < 64 else -1)
        if len(want_slots) >= total or after[b] == MOST:
            break
    want_slots = (want_slots + [-1] * total)[:total]
    assert slots.tolist() == want_slots


def test_pages_of_a_step():
    wide = dict(TABLE, batch=1 << 10, table_rows=1 << 10, max_pages=(1 << 20) + 1, page_table_row_stride=1 << 21)
    assert capi.update_page_table(**wide) == capi.FA_EINVAL and "2^30 pages" in capi.last_error()
