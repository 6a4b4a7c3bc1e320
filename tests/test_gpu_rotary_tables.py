"""rotary_cos_sin near the zeros of cosine and sine, where an error that is small beside 1 is not small beside the value."""
import pytest
import torch

import flash_attn_npu_v3 as fa
from oracle import fa_rotary_oracle as ro

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("table", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("how", [dict(), dict(base=500000.0, scaling="linear", factor=2.5)])
def test_near_zeros(how, table):
    """Multiples of a quarter turn are within 1e-5 of 355 / 2 k for f_0 = 1, and runs of positions cross the zeros of the slower
    angles. The angle is off by p f 2^-50 at most, as a whole; what is left of it after whole quarter turns keeps
    its bits, so sine and cosine are good to 2 steps of fp32 of the value (2^-22), the product by attention_factor and the rounding to
    the type to half a step each."""
    print(f"case table zeros {how} {table}", flush=True)
    dt, att, rd = TYPES[table], 1.25, 64
    pos = [11, 22, 33, 344, 355, 710, 1065, 52174, 103993, 104348, 208341, -355, 0] + list(range(1, 2000)) + list(range(130000, 131072, 3))
    got = fa.rotary_cos_sin(torch.tensor(pos, device=DEV), rd, attention_factor=att, dtype=dt, **how)
    f = torch.tensor(ro.frequencies(rd, **how), dtype=torch.float64)
    p = torch.tensor(pos, dtype=torch.float64)[:, None]
    least = 1.0
    for y, ref in zip(got, ro.table(pos, rd, attention_factor=att, **how)):
        half = torch.finfo(dt).eps / 2
        bound = att * (p * f).abs() * 2.0 ** -50 + ref.abs() * (2.0 ** -22 + 2.0 ** -24 + half) + torch.finfo(dt).smallest_normal * half
        off = (y.cpu().double() - ref).abs()
        assert (off <= bound).all(), (off / bound).max().item()
        least = min(least, ref[ref != 0].abs().min().item())
    assert least < 2e-5  # there are such values


def test_positions_past_all_bits():
    """Of a position of 2^55 or more 64 bits hold no part of a turn; cosines and sines still are such."""
    print("case table farthest", flush=True)
    pos = torch.tensor([2 ** 55, 2 ** 60 + 12345, 2 ** 63 - 1, -2 ** 63], device=DEV)
    c, s = fa.rotary_cos_sin(pos, 64, base=3.0)
    assert ((c.double() ** 2 + s.double() ** 2 - 1).abs() < 2.0 ** -20).all()
