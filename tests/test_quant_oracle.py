"""The 64-bit definitions of the quantised cache's operators (oracle/
fa_quant_oracle.py) against small cases worked by hand and against torch's own
e4m3 rounding. CPU only."""
import math

import pytest
import torch

from oracle import fa_quant_oracle as qo

E4M3 = torch.float8_e4m3fn


def test_page_table_step_by_hand():
    # pages of 4: request 0 grows over a page border, 1 ends, 2 is taken back by a page, 3 is new
    table = [[7, 0, 0], [3, 5, 0], [1, 2, 4], [0, 0, 0]]
    t, free, slots, cu, left = qo.page_table_step(table, [3, 6, 9, 0], [6, 0, 8, 5], [9, 8, 0, 0, 0, 0], 2, 4, 9)
    # freed in order: 3, 5 (request 1), 4 (request 2); stack 9 8 3 5 4, taken 4 (request 0), 5, 3 (request 3)
    assert free == [9, 8, 3, 5, 4, 0]
    assert t == [[7, 4, 0], [3, 5, 0], [1, 2, 4], [5, 3, 0]]
    assert slots == [7 * 4 + 3, 4 * 4, 4 * 4 + 1, 20, 21, 22, 23, 12, -1]
    assert cu == [0, 3, 3, 3, 8] and left == 2


def test_page_table_step_runs_empty():
    t, _, slots, cu, left = qo.page_table_step([[0, 0], [0, 0]], [0, 0], [3, 2], [6], 1, 2, 5)
    assert t == [[6, -1], [-1, 0]] and slots == [12, 13, -1, -1, -1] and cu == [0, 3, 5] and left == -2


def test_encode_e4m3_is_torch_rounding():
    x = torch.cat([torch.linspace(-448, 448, 4001), torch.linspace(-0.03, 0.03, 4001)]).double()
    assert torch.equal(qo.encode(x, E4M3).view(torch.uint8), x.float().to(E4M3).view(torch.uint8))


@pytest.mark.parametrize("dtype,top", [(torch.int8, 127.0), (E4M3, 448.0)])
def test_append_scale_is_the_smallest_power_of_two(dtype, top):
    for most, want in ((top, 1.0), (top * 1.01, 2.0), (top / 2, 0.5), (0.0, 2.0 ** -100), (top * 2.0 ** -101, 2.0 ** -100)):
        cache, scale = torch.zeros(1, 16, 1, 16).to(dtype), torch.zeros(1, 1, 1)
        x = torch.zeros(1, 1, 16, dtype=torch.float64)
        x[0, 0, 3] = -most
        qo.append(x, cache, scale, [0])
        assert scale.item() == want


def test_append_into_a_begun_block():
    cache, scale = torch.zeros(1, 32, 1, 16, dtype=torch.int8), torch.tensor([[[0.5], [4.0]]])
    cache[0, 0] = 101
    x = torch.full((2, 1, 16), 100.0, dtype=torch.bfloat16)
    qo.append(x, cache, scale, [1, 17])
    # 100 <= 127 * 1: the first block moves from 0.5 to 1 (101 * 0.5 = 50.5, to even 50), the second keeps 4
    assert scale.flatten().tolist() == [1.0, 4.0]
    assert cache[0, 0, 0, 0] == 50 and cache[0, 1, 0, 0] == 100 and cache[0, 17, 0, 0] == 25


def test_append_of_infinities_and_nan():
    x = torch.tensor([math.inf, -math.inf, math.nan, 1.0] * 4, dtype=torch.float16).view(1, 1, 16)
    for dtype in (torch.int8, E4M3):
        cache, scale = torch.zeros(1, 16, 1, 16).to(dtype), torch.zeros(1, 1, 1)
        qo.append(x, cache, scale, [3])
        y = cache[0, 3, 0].double() * scale.item()
        # s = 1024 (127 * 512 < 65504) and 256 (448 * 128 < 65504): 1 is 2^-10 of a code in int8 and 2^-8 in e4m3
        assert y[0].item() == 65536 and y[1] == -y[0] and y[3] == (0 if dtype == torch.int8 else 1)
        assert cache[0, 3, 0, 2].float() == 0 if dtype == torch.int8 else math.isnan(cache[0, 3, 0, 2].float())


def test_attend_by_hand():
    q = torch.tensor([[[1.0, 0.0]], [[0.0, 2.0]]])
    k = torch.tensor([[[1.0, 1.0]], [[3.0, 0.0]]]).double()
    v = torch.tensor([[[1.0, 0.0]], [[0.0, 1.0]]]).double()
    out, lse = qo.attend(q, k, v, torch.tensor([True, True]), 1.0, causal=True)
    assert out[0, 0].tolist() == [1.0, 0.0] and lse[0, 0].item() == 1.0
    w = 1 / (1 + math.exp(-2.0))
    assert abs(out[1, 0, 0].item() - w) < 1e-15 and abs(lse[0, 1].item() - math.log(math.exp(2) + 1)) < 1e-14
    out, lse = qo.attend(q, k, v, torch.tensor([False, False]), 1.0)
    assert not out.any() and torch.isinf(lse).all()
