"""torch.library.opcheck on the operators of the 4-bit cache, the read and the rotation: mutation and aliasing in their
schemas, meta shapes, tracing."""
import pytest
import torch

from fa_mi355x import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
UTILS = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")


def cache():
    g = torch.Generator().manual_seed(121)
    mk = lambda w, lo, hi: torch.randint(lo, hi, (6, 32, 2, w), generator=g, dtype=torch.uint8).to(DEV)  # noqa: E731
    return [mk(32, 0, 256), mk(32, 0, 256), mk(2, 120, 130), mk(2, 120, 130)]


def test_append():
    print("case opcheck fp4 append", flush=True)
    k, v = (torch.randn(5, 2, 64, device=DEV).to(torch.bfloat16) for _ in range(2))
    torch.library.opcheck(ops.quant_append, (k, v, *cache(), torch.tensor([33, 34, -1, 64, 65], device=DEV)), test_utils=UTILS)


@pytest.mark.parametrize("ragged", [False, True])
def test_fwd(ragged):
    print(f"case opcheck fp4 fwd {ragged}", flush=True)
    table, lens = torch.tensor([[1, 2], [4, 5]], **I32), torch.tensor([50, 33], **I32)
    q = torch.randn(2, 3, 4, 64, device=DEV).to(torch.float16)
    cu = torch.tensor([0, 2, 6], **I32) if ragged else None
    q = q.flatten(0, 1) if ragged else q
    torch.library.opcheck(ops.quant_fwd, (q, *cache(), lens, table, None, cu, 4 if ragged else 0, 0.125, True, -1, 0, 0.0), test_utils=UTILS)


def test_read():
    print("case opcheck read", flush=True)
    slots = torch.tensor([33, -1, 64], device=DEV)
    torch.library.opcheck(ops.quant_read, (*cache(), slots, None, 0, None, None, torch.float32), test_utils=UTILS)
    table, cu = torch.tensor([[1, 2], [4, 5]], **I32), torch.tensor([0, 40, 45], **I32)
    torch.library.opcheck(ops.quant_read, (*cache(), None, cu, 47, table, torch.tensor([1, 0], **I32), torch.bfloat16), test_utils=UTILS)


def test_rotary():
    print("case opcheck rotary", flush=True)
    pos = torch.tensor([3, 0, 7], device=DEV)
    torch.library.opcheck(ops.rotary_table, (pos, 32, 1e4, 3, 2.0, 100.0, 1.0, 32.0, 1.1, torch.float32), test_utils=UTILS)
    cos, sin = torch.rand(9, 16, device=DEV), torch.rand(9, 16, device=DEV)
    q, k = torch.randn(2, 3, 4, 64, device=DEV).to(torch.bfloat16), torch.randn(2, 3, 1, 64, device=DEV).to(torch.bfloat16)
    for kk in (k, None):
        for op in (ops.rotary, ops.rotary_):
            torch.library.opcheck(op, (q, kk, cos, sin, None, None, 2, None, True, False), test_utils=UTILS)
    torch.library.opcheck(ops.rotary, (q[0], None, cos, sin, None, torch.tensor([1], **I32), 0, torch.tensor([0, 2], **I32), False, True), test_utils=UTILS)
