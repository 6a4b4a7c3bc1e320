"""torch.library.opcheck on the operators of the quantised cache: mutation and aliasing in their schemas, meta
shapes, tracing; and the page table step, append and attention under torch.compile's tracing."""
import pytest
import torch

from fa_mi355x import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = dict(dtype=torch.int32, device=DEV)
UTILS = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")
# torch implements no arithmetic on float8_e4m3fn, which the schema and AOT checks perform on inputs
UTILS_FP8 = ("test_faketensor",)


def cache(dt):
    g = torch.Generator().manual_seed(121)
    codes = [torch.randint(-100, 100, (6, 32, 2, 64), generator=g).to(torch.int8).to(DEV) for _ in range(2)]
    if dt == torch.float8_e4m3fn:
        codes = [c.float().to(dt) for c in codes]
    return [*codes, torch.full((6, 2, 2), 0.02, device=DEV), torch.full((6, 2, 2), 0.03, device=DEV)]


def test_update_page_table():
    print("case opcheck update_page_table", flush=True)
    table = torch.tensor([[0, 1, 0], [2, 0, 0], [3, 0, 0]], **I32)
    free = torch.tensor([4, 5, 6, 7, 0, 0], **I32)
    lens, new = torch.tensor([40, 3, 30], **I32), torch.tensor([0, 36, 33], **I32)
    args = (table, lens, new, free, torch.tensor([4], **I32), 32, 40)
    torch.library.opcheck(ops.update_page_table, args, test_utils=UTILS)
    torch.library.opcheck(ops.update_page_table, args, dict(cache_batch_idx=torch.tensor([2, 0, 1], **I32)), test_utils=UTILS)


@pytest.mark.parametrize("dt", [torch.int8, torch.float8_e4m3fn])
def test_quant_append(dt):
    print(f"case opcheck quant_append {dt}", flush=True)
    k, v = (torch.randn(5, 2, 64, device=DEV).to(torch.bfloat16) for _ in range(2))
    slots = torch.tensor([33, 34, -1, 64, 65], device=DEV)
    torch.library.opcheck(ops.quant_append, (k, v, *cache(dt), slots), test_utils=UTILS if dt == torch.int8 else UTILS_FP8)


@pytest.mark.parametrize("dt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("ragged", [False, True])
def test_quant_fwd(dt, ragged):
    print(f"case opcheck quant_fwd {dt} {ragged}", flush=True)
    table, lens = torch.tensor([[1, 2], [4, 5]], **I32), torch.tensor([50, 33], **I32)
    q = torch.randn(2, 3, 4, 64, device=DEV).to(torch.float16)
    cu = torch.tensor([0, 2, 6], **I32) if ragged else None
    q = q.flatten(0, 1) if ragged else q
    args = (q, *cache(dt), lens, table, None, cu, 4 if ragged else 0, 0.125, True, -1, 0, 0.0)
    torch.library.opcheck(ops.quant_fwd, args, test_utils=UTILS if dt == torch.int8 else UTILS_FP8)
    args = (q, *cache(dt), lens, None, torch.tensor([3, 0], **I32), cu, 4 if ragged else 0, 0.125, False, 9, 1, 20.0)
    lens.clamp_(max=32)
    torch.library.opcheck(ops.quant_fwd, args, test_utils=UTILS if dt == torch.int8 else UTILS_FP8)
