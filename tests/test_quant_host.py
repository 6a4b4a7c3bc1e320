"""Refusals and shapes of the quantised cache's entry points, without a GPU: the C
entries' checks through ctypes, the struct mirrors, the operators' meta shapes."""
import ctypes
import os
import subprocess

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(REPO, "include", "fa_mi355x.h")
PTR = 1 << 20  # an aligned stand-in address: the checks never follow it

from fa_mi355x import capi  # noqa: E402


@pytest.mark.parametrize("struct,mirror", [("fa_page_table_params", capi.PageTableParams),
                                           ("fa_quant_append_params", capi.QuantAppendParams),
                                           ("fa_quant_fwd_params", capi.QuantFwdParams)])
def test_params_layout_matches_header(tmp_path, struct, mirror):
    names = [n for n, _ in mirror._fields_]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(['#include <stdio.h>', '#include <stddef.h>', '#include "fa_mi355x.h"', "int main(void) {",
                              f'  printf("size %zu\\n", sizeof({struct}));'] +
                             [f'  printf("{n} %zu\\n", offsetof({struct}, {n}));' for n in names] + ["  return 0; }"]))
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(mirror)
    for n in names:
        assert int(got[n]) == getattr(mirror, n).offset, n


CACHE = dict(k=PTR, k_page_stride=64 * 2 * 128, k_row_stride=2 * 128, k_head_stride=128,
             v=PTR, v_page_stride=64 * 2 * 128, v_row_stride=2 * 128, v_head_stride=128,
             k_scale=PTR, k_scale_page_stride=8, k_scale_block_stride=2, k_scale_head_stride=1,
             v_scale=PTR, v_scale_page_stride=8, v_scale_block_stride=2, v_scale_head_stride=1)
FWD = dict(dtype=1, cache_dtype=4, batch=2, seqlen_q=1, nheads=8, nheads_k=2, headdim=128, num_pages=9, page_size=64,
           scale_block=16, q=PTR, q_batch_stride=1024, q_row_stride=1024, q_head_stride=128, **CACHE, out=PTR,
           out_batch_stride=1024, out_row_stride=1024, out_head_stride=128, softmax_lse=PTR, cache_seqlens=PTR,
           page_table=PTR, page_table_row_stride=4, table_rows=2, max_pages=4, softmax_scale=0.1)


def test_fwd_accepts():
    assert capi.quant_fwd_workspace_size(capi.new_quant_fwd_params(**FWD))[0] == capi.FA_OK
    for more in (dict(cache_dtype=3), dict(dtype=0), dict(headdim=16), dict(page_table=None, num_pages=2),
                 dict(seqlen_q=0, q=None, out=None, softmax_lse=None), dict(cu_seqlens_q=PTR, total_q=0, q=None),
                 dict(window_size_left=2 ** 31 - 1), dict(table_rows=1, cache_batch_idx=PTR)):
        p = capi.new_quant_fwd_params(**dict(FWD, **more))
        assert capi.quant_fwd_workspace_size(p)[0] == capi.FA_OK, (more, capi.last_error())


@pytest.mark.parametrize("more,says", [
    (dict(abi_version=3), "abi_version"), (dict(dtype=3), "fp16 and bf16"), (dict(dtype=2), "fp16 and bf16"),
    (dict(cache_dtype=1), "int8 or float8_e4m3fn"), (dict(headdim=120), "multiple of 16"),
    (dict(headdim=272), "multiple of 16"), (dict(headdim=0), "multiple of 16"), (dict(nheads=7), "divide"),
    (dict(nheads=0), "divide"), (dict(nheads_k=0), "key/value heads"), (dict(batch=0), "batch"),
    (dict(seqlen_q=-1), "negative"), (dict(scale_block=8), "multiple of 16 tokens"),
    (dict(scale_block=24), "multiple of 16 tokens"), (dict(page_size=72), "multiple of the 16 tokens"),
    (dict(page_size=0), "multiple of the 16 tokens"), (dict(softcap=-1.0), "softcap"), (dict(cache_seqlens=None), "cache_seqlens"),
    (dict(num_pages=0), "a page"), (dict(table_rows=1), "row per sequence"), (dict(max_pages=0), "rows and columns"),
    (dict(max_pages=1 << 26), "2^31"), (dict(page_table=None, num_pages=1), "row per sequence"), (dict(q=None), "required"),
    (dict(v_scale=None), "required"), (dict(softmax_lse=None), "required"), (dict(q=PTR + 8), "aligned"), (dict(k=PTR + 4), "aligned"),
    (dict(q_row_stride=1028), "multiples of 8"), (dict(out_head_stride=4), "multiples of 8"),
    (dict(k_row_stride=264), "multiples of 16"), (dict(v_head_stride=8), "multiples of 16"),
    (dict(seqlen_q=1 << 30), "too many query rows"), (dict(k_row_stride=1 << 27), "row strides"),
    (dict(v_row_stride=-256), "row strides")])
def test_fwd_refuses(more, says):
    p = capi.new_quant_fwd_params(**dict(FWD, **more))
    assert capi.quant_fwd(p) == capi.FA_EINVAL and says in capi.last_error(), capi.last_error()


APPEND = dict(dtype=1, cache_dtype=4, nheads_k=2, headdim=128, num_pages=9, page_size=64, scale_block=16, total_new=5,
              k_new=PTR, knew_row_stride=256, knew_head_stride=128, v_new=PTR, vnew_row_stride=256, vnew_head_stride=128,
              **CACHE, slot_mapping=PTR)


def test_append_of_nothing():
    assert capi.quant_append(**dict(APPEND, total_new=0, k_new=None, slot_mapping=None)) == capi.FA_OK


@pytest.mark.parametrize("more,says", [
    (dict(dtype=3), "fp16 and bf16"), (dict(cache_dtype=0), "int8 or float8_e4m3fn"), (dict(headdim=8), "multiple of 16"),
    (dict(page_size=40), "multiple of the 16 tokens"), (dict(scale_block=0), "multiple of 16 tokens"), (dict(nheads_k=70000), "key/value heads"),
    (dict(total_new=-1), "new rows"), (dict(total_new=1 << 31), "new rows"), (dict(k_new=None), "required"), (dict(slot_mapping=None), "required"),
    (dict(v_new=PTR + 2), "aligned"), (dict(knew_row_stride=1 << 24), "row strides"), (dict(knew_row_stride=260), "multiples of 8"), (dict(v_page_stride=8), "multiples of 16")])
def test_append_refuses(more, says):
    assert capi.quant_append(**dict(APPEND, **more)) == capi.FA_EINVAL and says in capi.last_error(), capi.last_error()


TABLE = dict(batch=2, page_size=16, table_rows=2, max_pages=4, page_table=PTR, page_table_row_stride=4, cache_seqlens=PTR,
             new_seqlens=PTR, free_pages=PTR, free_capacity=8, num_free=PTR, num_free_out=PTR, cu_seqlens_new=PTR,
             slot_mapping=PTR, total_new=2)


@pytest.mark.parametrize("more,says", [
    (dict(batch=0), "batch"), (dict(page_size=0), "page_size"), (dict(table_rows=1), "row per request"),
    (dict(max_pages=1 << 28), "2^31"), (dict(page_table=None), "page_table"), (dict(page_table_row_stride=3), "overlap"),
    (dict(free_capacity=-1), "free_pages"), (dict(free_pages=None), "free_pages"), (dict(num_free=None), "required"),
    (dict(cu_seqlens_new=None), "required"), (dict(total_new=-1), "total_new"), (dict(total_new=1 << 31), "total_new"), (dict(slot_mapping=None), "slot_mapping")])
def test_page_table_refuses(more, says):
    assert capi.update_page_table(**dict(TABLE, **more)) == capi.FA_EINVAL and says in capi.last_error(), capi.last_error()


def test_null_params():
    for fn in ("fa_update_page_table", "fa_quant_append", "fa_quant_fwd"):
        assert getattr(capi.lib(), fn)(None, None) == capi.FA_EINVAL
    n = ctypes.c_size_t(0)
    assert capi.lib().fa_quant_fwd_workspace_size(None, ctypes.byref(n)) == capi.FA_EINVAL
    p = capi.new_quant_fwd_params(**FWD)
    assert capi.lib().fa_quant_fwd_workspace_size(ctypes.byref(p), None) == capi.FA_EINVAL


def test_workspace_is_asked_for():
    p = capi.new_quant_fwd_params(**FWD)
    st, n = capi.quant_fwd_workspace_size(p)
    if n:
        assert capi.quant_fwd(p) == capi.FA_EWORKSPACE
        p.workspace, p.workspace_bytes = PTR, n - 1
        assert capi.quant_fwd(p) == capi.FA_EWORKSPACE
        p.workspace, p.workspace_bytes = PTR + 16, n
        assert capi.quant_fwd(p) == capi.FA_EWORKSPACE


def test_meta_shapes_and_no_cpu_path():
    import flash_attn_npu_v3 as fa
    for dev in ("meta", "cpu"):
        mk = lambda *s, dt=torch.bfloat16: torch.zeros(s, device=dev).to(dt)  # noqa: E731
        kc, vc, ks, vs = mk(9, 64, 2, 128, dt=torch.int8), mk(9, 64, 2, 128, dt=torch.int8), mk(9, 4, 2, dt=torch.float32), \
            mk(9, 4, 2, dt=torch.float32)
        lens, table = mk(2, dt=torch.int32), mk(2, 4, dt=torch.int32)
        calls = (lambda: fa.flash_attn_with_quantized_kvcache(mk(2, 3, 8, 128), kc, vc, ks, vs, lens, page_table=table,
                                                              return_softmax_lse=True),
                 lambda: fa.append_quantized_kvcache(mk(5, 2, 128), mk(5, 2, 128), kc, vc, ks, vs, mk(5, dt=torch.int64)),
                 lambda: fa.update_page_table(table, lens, lens, lens, lens[:1], 64, 7))
        if dev == "cpu":
            for call in calls:
                with pytest.raises((NotImplementedError, RuntimeError)):
                    call()
            continue
        out, lse = calls[0]()
        assert out.shape == (2, 3, 8, 128) and out.dtype == torch.bfloat16 and lse.shape == (2, 8, 3) and lse.dtype == torch.float32
        assert calls[1]() is None
        slots, cu, left = calls[2]()
        assert slots.shape == (7,) and slots.dtype == torch.int64 and cu.shape == (3,) and left.shape == (1,)
    q = torch.zeros(4, 8, 128)
    with pytest.raises(RuntimeError, match="max_seqlen_q"):
        fa.flash_attn_with_quantized_kvcache(q, q, q, q, q, q, cu_seqlens_q=q)
