"""Refusals and shapes of the 4-bit cache's, the read's and the rotary entry points, without a GPU: the C entries' checks
through ctypes, the struct mirrors, the operators' meta shapes, the oracles against torch."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from fa_mi355x import capi
from oracle import fa_fp4_oracle as fo
from oracle import fa_rotary_oracle as ro
from tests.test_quant_host import HEADER, PTR, REPO
from tests.test_quant_sanitize import CSRC, HOST, build_and_run


@pytest.mark.parametrize("struct,mirror", [("fa_quant_read_params", capi.QuantReadParams), ("fa_rotary_table_params", capi.RotaryTableParams),
                                           ("fa_rotary_params", capi.RotaryParams)])
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


ROW = 2 * 64  # bytes of a row of two heads of 128 channels
CACHE = dict(k=PTR, k_page_stride=64 * ROW, k_row_stride=ROW, k_head_stride=64, v=PTR, v_page_stride=64 * ROW, v_row_stride=ROW,
             v_head_stride=64, k_scale=PTR + 1, k_scale_page_stride=64 * 8, k_scale_block_stride=8, k_scale_head_stride=4,
             v_scale=PTR + 3, v_scale_page_stride=64 * 8, v_scale_block_stride=8, v_scale_head_stride=4)
FWD = dict(dtype=1, cache_dtype=5, batch=2, seqlen_q=1, nheads=8, nheads_k=2, headdim=128, num_pages=9, page_size=64,
           scale_block=1, q=PTR, q_batch_stride=1024, q_row_stride=1024, q_head_stride=128, **CACHE, out=PTR,
           out_batch_stride=1024, out_row_stride=1024, out_head_stride=128, softmax_lse=PTR, cache_seqlens=PTR,
           page_table=PTR, page_table_row_stride=4, table_rows=2, max_pages=4, softmax_scale=0.1)


def test_fwd_accepts():
    for more in (dict(), dict(dtype=0), dict(headdim=32), dict(page_table=None, num_pages=2), dict(page_size=16), dict(page_size=48),
                 dict(seqlen_q=0, q=None, out=None, softmax_lse=None), dict(cu_seqlens_q=PTR, total_q=0, q=None),
                 dict(max_pages=1 << 24, page_table_row_stride=1 << 24)):
        p = capi.new_quant_fwd_params(**dict(FWD, **more))
        assert capi.fp4_fwd_workspace_size(p)[0] == capi.FA_OK, (more, capi.last_error())


@pytest.mark.parametrize("more,says", [
    (dict(abi_version=3), "abi_version"), (dict(dtype=5), "fp16 and bf16"), (dict(cache_dtype=4), "float4_e2m1"), (dict(cache_dtype=3), "float4_e2m1"),
    (dict(headdim=48), "multiple of 32"), (dict(headdim=288), "multiple of 32"), (dict(headdim=0), "multiple of 32"), (dict(nheads=7), "divide"),
    (dict(scale_block=16), "scales of its own"), (dict(page_size=8), "multiple of 16"), (dict(page_size=24), "multiple of 16"),
    (dict(page_size=0), "multiple of 16"), (dict(k_row_stride=136), "multiples of 16"), (dict(v=PTR + 8), "aligned"), (dict(k_scale=None), "required"),
    (dict(max_pages=(1 << 24) + 1, page_table_row_stride=1 << 25), "2^30 tokens"), (dict(num_pages=0), "page"), (dict(cache_seqlens=None), "cache_seqlens")])
def test_fwd_refuses(more, says):
    p = capi.new_quant_fwd_params(**dict(FWD, **more))
    assert capi.fp4_fwd_workspace_size(p)[0] == capi.FA_EINVAL and says in capi.last_error(), capi.last_error()
    assert capi.fp4_fwd(p) == capi.FA_EINVAL


def test_the_entries_keep_to_their_caches():
    p = capi.new_quant_fwd_params(**FWD)
    assert capi.quant_fwd_workspace_size(p)[0] == capi.FA_EINVAL and capi.quant_fwd(p) == capi.FA_EINVAL
    assert capi.quant_append(**APPEND) == capi.FA_EINVAL


def test_workspace_is_asked_for():
    p = capi.new_quant_fwd_params(**FWD)
    st, n = capi.fp4_fwd_workspace_size(p)
    assert st == capi.FA_OK and n > 0
    assert capi.fp4_fwd(p) == capi.FA_EWORKSPACE
    p.workspace, p.workspace_bytes = PTR, n - 1
    assert capi.fp4_fwd(p) == capi.FA_EWORKSPACE
    p.workspace, p.workspace_bytes = PTR + 16, n
    assert capi.fp4_fwd(p) == capi.FA_EWORKSPACE


APPEND = dict(dtype=1, cache_dtype=5, nheads_k=2, headdim=128, num_pages=9, page_size=64, scale_block=1, total_new=3, k_new=PTR,
              knew_row_stride=256, knew_head_stride=128, v_new=PTR, vnew_row_stride=256, vnew_head_stride=128, slot_mapping=PTR, **CACHE)


@pytest.mark.parametrize("more,says", [
    (dict(dtype=2), "fp16 and bf16"), (dict(cache_dtype=3), "float4_e2m1"), (dict(headdim=80), "multiple of 32"), (dict(scale_block=16), "scales of its own"),
    (dict(total_new=-1), "new rows"), (dict(total_new=1 << 31), "new rows"), (dict(k_new=None), "required"), (dict(v_scale=None), "required"),
    (dict(v_new=PTR + 2), "aligned"), (dict(knew_row_stride=260), "multiples of 8"), (dict(knew_row_stride=1 << 24), "row strides"),
    (dict(k_head_stride=8), "multiples of 16"), (dict(nheads_k=0), "key/value heads")])
def test_append_refuses(more, says):
    assert capi.fp4_append(**dict(APPEND, **more)) == capi.FA_EINVAL and says in capi.last_error(), capi.last_error()


READ = dict(dtype=1, cache_dtype=5, nheads_k=2, headdim=128, num_pages=9, page_size=64, scale_block=1, total=3, k_out=PTR, v_out=PTR,
            cu_seqlens_k=PTR, batch=2, page_table=PTR, page_table_row_stride=4, table_rows=2, max_pages=4, **CACHE)


@pytest.mark.parametrize("more,says", [
    (dict(dtype=3), "fp32, fp16 or bf16"), (dict(cache_dtype=1), "int8 or float8_e4m3fn"), (dict(cache_dtype=4), "multiple of 16 tokens"),
    (dict(headdim=80), "multiple of 32"), (dict(total=-1), "rows"), (dict(total=1 << 31), "rows"), (dict(k_out=None), "required"), (dict(v_out=PTR + 8), "aligned"),
    (dict(slot_mapping=PTR), "either"), (dict(cu_seqlens_k=None), "either"), (dict(batch=0), "batch"), (dict(table_rows=1), "row per sequence"),
    (dict(max_pages=0), "rows and columns"), (dict(page_table=None, batch=10), "row per sequence"), (dict(v=None), "required"),
    (dict(k_page_stride=8), "multiples of 16"), (dict(k=PTR + 4), "aligned")])
def test_read_refuses(more, says):
    assert capi.quant_read(**dict(READ, **more)) == capi.FA_EINVAL and says in capi.last_error(), capi.last_error()


TABLE = dict(dtype=2, rotary_dim=64, scaling=0, base=1e4, factor=1.0, attention_factor=1.0, num_positions=4, positions=PTR, cos=PTR, sin=PTR)


@pytest.mark.parametrize("more,says", [
    (dict(dtype=3), "fp32, fp16 or bf16"), (dict(rotary_dim=8), "multiple of 16"), (dict(rotary_dim=272), "multiple of 16"), (dict(rotary_dim=-16), "multiple of 16"),
    (dict(num_positions=-1), "negative"), (dict(base=-1.0), "base"), (dict(base=float("inf")), "base"), (dict(factor=float("nan")), "factor"), (dict(scaling=4), "scaling"),
    (dict(scaling=-1), "scaling"), (dict(scaling=3), "original_length"), (dict(scaling=3, original_length=8.0), "low"), (dict(cos=None), "required"),
    (dict(scaling=1, factor=5e-324, base=1e-300), "not finite"), (dict(sin=PTR + 8), "aligned"), (dict(attention_factor=float("nan")), "attention_factor")])
def test_table_refuses(more, says):
    assert capi.rotary_table(**dict(TABLE, **more)) == capi.FA_EINVAL and says in capi.last_error(), capi.last_error()


def rows(*names, b=2048, i=512, h=64):
    f = {}
    for n in names:
        f.update({n: PTR if "out" not in n else 2 * PTR, n + "_batch_stride": b, n + "_row_stride": i, n + "_head_stride": h})
    return f


ROTARY = dict(dtype=1, table_dtype=2, batch=2, seqlen=4, nheads=8, nheads_k=2, headdim=64, rotary_dim=32, **rows("q", "k", "q_out", "k_out"),
              cos=PTR, cos_row_stride=16, sin=PTR, sin_row_stride=16, seqlen_ro=9)


@pytest.mark.parametrize("more,says", [
    (dict(dtype=2), "fp16 and bf16"), (dict(table_dtype=0), "dtype of q"), (dict(rotary_dim=24), "multiple of 16"), (dict(rotary_dim=80), "exceeds"),
    (dict(headdim=60), "multiple of 8"), (dict(nheads=0), "heads"), (dict(nheads_k=-1), "heads"), (dict(nheads_k=65536), "heads"), (dict(batch=-1), "negative"),
    (dict(batch=1 << 16, seqlen=1 << 16), "2^31 rows"), (dict(cu_seqlens=PTR, batch=0, total=3), "sequence"), (dict(seqlen_ro=0), "row"), (dict(q=None), "required"),
    (dict(k_out=None), "required"), (dict(q_out=PTR), "neither"), (dict(q_out=PTR, k_out=PTR, q_out_row_stride=520), "strides of q and k"), (dict(q=PTR + 8), "aligned"),
    (dict(k_head_stride=60), "multiples of 8"), (dict(cos_row_stride=20), "multiples of 8"), (dict(cos=PTR + 4), "aligned"), (dict(headdim=65536, nheads=65535), "too many heads")])
def test_rotary_refuses(more, says):
    assert capi.rotary(**dict(ROTARY, **more)) == capi.FA_EINVAL and says in capi.last_error(), capi.last_error()


def test_nothing_to_do():
    assert capi.rotary(**dict(ROTARY, batch=0, q=None, k=None, cos=None)) == capi.FA_OK
    assert capi.rotary_table(**dict(TABLE, num_positions=0, positions=None, cos=None, sin=None)) == capi.FA_OK
    assert capi.quant_read(**dict(READ, total=0, k_out=None, v_out=None)) == capi.FA_OK
    assert capi.fp4_append(**dict(APPEND, total_new=0, k_new=None)) == capi.FA_OK


def test_null_params():
    for fn in ("fa_fp4_append", "fa_fp4_fwd", "fa_quant_read", "fa_rotary_table", "fa_rotary"):
        assert getattr(capi.lib(), fn)(None, None) == capi.FA_EINVAL
    n = ctypes.c_size_t(0)
    assert capi.lib().fa_fp4_fwd_workspace_size(None, ctypes.byref(n)) == capi.FA_EINVAL
    p = capi.new_quant_fwd_params(**FWD)
    assert capi.lib().fa_fp4_fwd_workspace_size(ctypes.byref(p), None) == capi.FA_EINVAL


def test_meta_shapes_and_no_cpu_path():
    import flash_attn_npu_v3 as fa
    for dev in ("meta", "cpu"):
        mk = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device=dev)  # noqa: E731
        u8, i32 = torch.uint8, torch.int32
        cache = mk(9, 64, 2, 64, dt=u8), mk(9, 64, 2, 64, dt=u8), mk(9, 64, 2, 4, dt=u8), mk(9, 64, 2, 4, dt=u8)
        lens, table = mk(2, dt=i32), mk(2, 4, dt=i32)
        calls = (lambda: fa.flash_attn_with_quantized_kvcache(mk(2, 3, 8, 128), *cache, lens, page_table=table, return_softmax_lse=True),
                 lambda: fa.append_quantized_kvcache(mk(5, 2, 128), mk(5, 2, 128), *cache, mk(5, dt=torch.int64)),
                 lambda: fa.read_quantized_kvcache(*cache, cu_seqlens_k=mk(3, dt=i32), total_k=11, page_table=table, dtype=torch.float16),
                 lambda: fa.rotary_cos_sin(mk(7, dt=i32), 32, dtype=torch.float16),
                 lambda: fa.apply_rotary_emb(mk(2, 3, 8, 128), mk(2, 3, 1, 128), mk(9, 16), mk(9, 16)),
                 lambda: fa.apply_rotary_emb(mk(3, 8, 128), None, mk(9, 16), mk(9, 16), inplace=True))
        if dev == "cpu":
            for call in calls:
                with pytest.raises((NotImplementedError, RuntimeError)):
                    call()
            continue
        out, lse = calls[0]()
        assert out.shape == (2, 3, 8, 128) and lse.shape == (2, 8, 3) and lse.dtype == torch.float32
        assert calls[1]() is None
        assert all(t.shape == (11, 2, 128) and t.dtype == torch.float16 for t in calls[2]())
        assert all(t.shape == (7, 16) and t.dtype == torch.float16 for t in calls[3]())
        q, k = calls[4]()
        assert q.shape == (2, 3, 8, 128) and k.shape == (2, 3, 1, 128)
        assert calls[5]().shape == (3, 8, 128)
    q = torch.zeros(4, 8, 128)
    with pytest.raises(RuntimeError, match="total_k"):
        fa.read_quantized_kvcache(q, q, q, q, cu_seqlens_k=q)
    with pytest.raises(RuntimeError, match="scaling"):
        fa.rotary_cos_sin(q, 32, scaling="dynamic")


def test_oracle_scales_and_codes():
    """The oracle's own borders: largest values keep finite, ties go to the even code, scales are the smallest."""
    for dt in (torch.bfloat16, torch.float16):
        big = torch.finfo(dt).max
        codes, byte = fo.group([big, -big] + [0.0] * 30, dt)
        assert codes[:2] == [7, 15] and byte == fo.HIGHEST[dt] + 127
        v = fo.values(torch.tensor([7 + 16 * 15] + [0] * 15, dtype=torch.uint8), torch.tensor([byte], dtype=torch.uint8))
        assert torch.isfinite(v.to(dt)).all()
        assert fo.group([math_nan()] + [1.0] * 31, dt)[1] == 255
        assert fo.group([0.0] * 32, dt)[1] == 27
    for x, code in ((0.25, 0), (0.75, 2), (1.25, 2), (1.75, 4), (2.5, 4), (3.5, 6), (5.0, 6), (6.0, 7)):
        assert fo.group([x, 6.0] + [0.0] * 30, torch.bfloat16)[0][0] == code
    assert fo.group([6.0] + [0.0] * 31, torch.bfloat16)[1] == 127 and fo.group([6.0625] + [0.0] * 31, torch.bfloat16)[1] == 128


def math_nan():
    return float("nan")


def test_oracle_rotation():
    """As multiplication of complex numbers, and back."""
    g = torch.Generator().manual_seed(1)
    cos, sin = ro.table(range(7), 32)
    x = torch.randn(7, 3, 48, generator=g, dtype=torch.float64)
    for inter in (True, False):
        y = ro.turn(x, cos, sin, inter)
        assert (ro.turn(y, cos, -sin, inter) - x).abs().max() < 1e-14 and torch.equal(y[..., 32:], x[..., 32:])
        pairs = torch.complex(*(x[..., i] for i in ((slice(0, 32, 2), slice(1, 32, 2)) if inter else (slice(0, 16), slice(16, 32)))))
        z = pairs * torch.polar(torch.ones(7, 16, dtype=torch.float64), torch.arange(7.0, dtype=torch.float64)[:, None] *
                                10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16))[:, None]
        got = torch.complex(*(y[..., i] for i in ((slice(0, 32, 2), slice(1, 32, 2)) if inter else (slice(0, 16), slice(16, 32)))))
        assert (got - z).abs().max() < 1e-13


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_checks_and_plans(tmp_path):
    """The host code with AddressSanitizer and UndefinedBehaviorSanitizer over recording stubs of the launchers."""
    build_and_run(tmp_path, "-D__HIP_PLATFORM_AMD__=1", "-I", "/opt/rocm/include", "-I", os.path.join(REPO, "include"),
                  os.path.join(CSRC, "fa_fp4_api.cpp"), os.path.join(CSRC, "fa_rotary_api.cpp"), os.path.join(HOST, "fa_fp4_host_harness.cpp"))
