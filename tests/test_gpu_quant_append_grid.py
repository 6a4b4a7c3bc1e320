"""Appends of more units (runs of rows x heads) than one launch has threads for."""
import pytest
import torch

import flash_attn_npu_v3 as fa

pytestmark = pytest.mark.gpu
DEV = "cuda"
HK, D = 65535, 16


def append(total, slots, page):
    """The same row again and again into a cache of `page` rows, read back as codes (page, HK, D) and scales (blocks, HK)."""
    g = torch.Generator().manual_seed(81)
    k, v = (torch.randn(1, HK, D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    kc, vc = (torch.full((1, page, HK, D), -7, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.full((1, page // 16, HK), 3.0, device=DEV) for _ in range(2))
    fa.append_quantized_kvcache(k.expand(total, HK, D), v.expand(total, HK, D), kc, vc, ks, vs, slots.to(DEV))
    out = []
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        most = x[0].abs().amax(-1).double()
        m, e = torch.frexp(most)  # 127 = 0.9921875 * 2^7
        # 2^e by its bits: pow is not exact on the GPU, and many x / scale lie half way between two codes
        scale = ((e.int() - 7 + (m > 127 / 128).int() + 127) << 23).view(torch.float32)
        out.append((c[0], s[0], torch.round(x[0].double() / scale.double()[:, None]).to(torch.int8), scale))
    return out


def test_few_rows():
    print("case append grid, few rows", flush=True)
    total = 600  # 600 x 131070 units of a wave
    slots = torch.full((total,), -1)
    at = [0, 1, 300, 511, 512, 513, 598, 599]
    slots[at] = torch.arange(len(at)) * 16  # a block each
    for codes, scales, want, scale in append(total, slots, 128):
        assert (codes[::16] == want).all() and (scales == scale).all()
        left = torch.ones(128, dtype=torch.bool)
        left[::16] = False
        assert (codes[left.to(DEV)] == -7).all()


def test_many_rows():
    """A run of every length across the ends of the launches."""
    print("case append grid, many rows", flush=True)
    total = 20000  # 1250 chunks of 16 rows: launches of 512 chunks
    slots = torch.full((total,), -1)
    runs = [(0, 16), (8185, 16), (8208, 3), (16383, 2), (16391, 16), (19984, 16)]
    for i, (first, n) in enumerate(runs):
        slots[first:first + n] = 16 * i + torch.arange(n)
    for codes, scales, want, scale in append(total, slots, 96):
        assert (scales == scale).all()
        for i, (_, n) in enumerate(runs):
            assert (codes[16 * i:16 * i + n] == want).all() and (codes[16 * i + n:16 * i + 16] == -7).all()
