"""CPU-side checks of the sparse paged operators' boundary: argument layouts, what the entry points refuse (with made-up pointers: nothing is launched), what the
Python functions refuse."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

from keys_values_amd import _lib
from keys_values_amd.attention import ops
from keys_values_amd.kvcache.paged import PagedKVCacheBuffers, paged_append, paged_bounds
from keys_values_amd.longctx import ops as rows

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "kvx.h")
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up: where nothing can be launched")
INVALID, UNSUPPORTED = _lib.KVX_ERR_INVALID, _lib.KVX_ERR_UNSUPPORTED


def test_struct_layouts_match_c(tmp_path):
    structs = {"kvx_paged_append_args": _lib.PagedAppendArgs, "kvx_paged_bounds_args": _lib.PagedBoundsArgs, "kvx_paged_select_args": _lib.PagedSelectArgs,
               "kvx_chosen_pages": _lib.ChosenPages}
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){"]
    for cname, cls in structs.items():
        src.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        src += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "layout.c").write_text("\n".join(src + ["return 0;}"]))
    subprocess.check_call(["gcc", "-std=c11", str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")])
    got = dict(line.split() for line in subprocess.check_output([str(tmp_path / "layout")], text=True).splitlines())
    for cname, cls in structs.items():
        assert int(got[cname]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(cls, f).offset, f"{cname}.{f}"


def _set(block, fields):
    for name, value in dict(fields).items():
        setattr(block, name, value)


def _pages(p, fields):
    p.num_pages, p.page_size, p.Hkv, p.D, p.kv_dtype = 100, 16, 2, 128, _lib.KVX_KV_BF16
    p.k = p.v = p.k_scale = p.k_zp = p.v_scale = p.v_zp = 4096
    p.k_stride_t = p.v_stride_t = 128
    p.k_stride_h = p.v_stride_h = 16 * 128
    p.k_stride_page = p.v_stride_page = 2 * 16 * 128
    p.qs_stride_h, p.qs_stride_page = 16, 32
    _set(p, fields)


def _append(kvx, pages=(), rotary=(), slots=4096):
    a = _lib.PagedAppendArgs()
    r = a.rotary
    r.qkv, r.stride_t, r.tokens, r.Hq, r.Hkv, r.D, r.rotary_dim, r.elem_dtype, r.table_rows = 4096, 12 * 128, 9, 8, 2, 128, 64, _lib.KVX_KV_BF16, 50
    r.cos = r.sin = r.positions = r.q_weight = r.k_weight = 4096
    _set(r, rotary)
    _pages(a.pages, pages)
    a.slots = slots
    return kvx.kvx_paged_append(ctypes.byref(a), None)


def _bounds(kvx, pages=(), **fields):
    a = _lib.PagedBoundsArgs()
    _pages(a.pages, pages)
    a.B, a.max_pages, a.tokens, a.block_table, a.bt_stride_b, a.lens, a.bounds = 3, 7, 40, 4096, 7, 4096, 4096
    a.b_stride_side, a.b_stride_h, a.b_stride_page = 128, 256, 512
    _set(a, fields)
    return kvx.kvx_paged_bounds(ctypes.byref(a), None)


def _select_args(**fields):
    a = _lib.PagedSelectArgs()
    a.num_pages, a.page_size, a.Hkv, a.D, a.elem_dtype, a.B, a.Hq, a.max_pages, a.count, a.first, a.last = 100, 16, 2, 128, _lib.KVX_KV_BF16, 3, 8, 70, 10, 1, 1
    a.q = a.bounds = a.block_table = a.lens = a.chosen = a.workspace = 4096
    a.q_stride_b, a.q_stride_h, a.bt_stride_b = 1024, 128, 70
    a.b_stride_side, a.b_stride_h, a.b_stride_page = 128, 256, 512
    a.workspace_bytes = 2**40
    _set(a, fields)
    return a


def _select(kvx, **fields):
    return kvx.kvx_paged_select(ctypes.byref(_select_args(**fields)), None)


def _decode_args(pages=(), chosen=(), **fields):
    a, c = _lib.PagedDecodeArgs(), _lib.ChosenPages()
    _pages(a.pages, pages)
    a.B, a.Hq, a.max_pages, a.sm_scale, a.q, a.block_table, a.lens, a.o, a.bt_stride_b = 3, 8, 200, 0.1, 4096, 4096, 4096, 4096, 200
    a.q_stride_b = a.o_stride_b = 8 * 128
    a.q_stride_h = a.o_stride_h = 128
    a.workspace, a.workspace_bytes = 4096, 2**40
    c.pages, c.stride_b, c.stride_h, c.count = 4096, 100, 50, 50
    _set(a, fields)
    _set(c, chosen)
    return a, c


def _decode(kvx, pages=(), chosen=(), **fields):
    return kvx.kvx_paged_decode_chosen(*(ctypes.byref(x) for x in _decode_args(pages, chosen, **fields)), None)


BAD_PAGES = [
    (dict(num_pages=0), INVALID), (dict(k=0), INVALID), (dict(v=4100), INVALID), (dict(k_stride_t=132), INVALID), (dict(v_stride_page=-4096), INVALID),
    (dict(page_size=8), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED), (dict(page_size=2048), UNSUPPORTED), (dict(kv_dtype=6), UNSUPPORTED), (dict(k_stride_t=64), UNSUPPORTED),
    (dict(k_stride_page=2**31), UNSUPPORTED), (dict(kv_dtype=_lib.KVX_KV_U8, k_scale=0), INVALID), (dict(kv_dtype=_lib.KVX_KV_U8, qs_stride_h=18), INVALID),
    (dict(D=96), UNSUPPORTED), (dict(Hkv=0), INVALID),
]


@no_device
@pytest.mark.parametrize("call", [_append, _bounds, _decode])
def test_pages_are_checked(kvx, call):
    for good in ({}, dict(kv_dtype=_lib.KVX_KV_U8), dict(kv_dtype=_lib.KVX_KV_U4, k_stride_t=64, v_stride_t=64), dict(page_size=1024)):
        assert call(kvx, good) == _lib.KVX_ERR_HIP, good  # no device
    for bad, status in BAD_PAGES:
        assert call(kvx, bad) == status, bad
        assert kvx.kvx_last_error()


@no_device
def test_append_is_checked(kvx):
    assert kvx.kvx_paged_append(None, None) == INVALID
    assert _append(kvx, rotary=dict(q_weight=0, k_weight=0)) == _append(kvx, rotary=dict(tokens=1, stride_t=0)) == _lib.KVX_ERR_HIP
    assert _append(kvx, rotary=dict(tokens=0, qkv=0), slots=0) == _lib.KVX_OK
    for bad in (dict(tokens=-1), dict(Hq=0), dict(Hkv=0), dict(qkv=0), dict(cos=0), dict(sin=4100), dict(positions=0), dict(q_weight=0), dict(k_weight=4100), dict(stride_t=12 * 128 - 8),
                dict(stride_t=12 * 128 + 4), dict(qkv=4104), dict(table_rows=0), dict(Hkv=1), dict(Hkv=3, stride_t=2048), dict(D=64), dict(elem_dtype=_lib.KVX_KV_F16)):
        assert _append(kvx, rotary=bad) == INVALID, bad
    assert _append(kvx, slots=0) == INVALID
    for bad in (dict(D=96), dict(rotary_dim=0), dict(rotary_dim=8), dict(rotary_dim=144), dict(elem_dtype=_lib.KVX_KV_U8), dict(Hq=65536), dict(tokens=2**31), dict(tokens=2**26)):
        assert _append(kvx, rotary=bad) == UNSUPPORTED, bad


@no_device
def test_bounds_are_checked(kvx):
    assert kvx.kvx_paged_bounds(None, None) == INVALID
    assert _bounds(kvx, tokens=2**31 - 1) == _lib.KVX_ERR_HIP
    assert _bounds(kvx, B=0) == _bounds(kvx, tokens=0, bounds=0) == _lib.KVX_OK
    for bad in (dict(B=-1), dict(max_pages=0), dict(tokens=-1), dict(block_table=0), dict(lens=0), dict(bounds=0), dict(bounds=4104), dict(b_stride_page=516), dict(b_stride_h=-256),
                dict(b_stride_side=4), dict(bt_stride_b=-1)):
        assert _bounds(kvx, **bad) == INVALID, bad
    for bad in (dict(B=65536), dict(max_pages=2**26), dict(B=60000, max_pages=2**20, tokens=2**20)):
        assert _bounds(kvx, **bad) == UNSUPPORTED, bad


@no_device
def test_select_is_checked(kvx):
    assert kvx.kvx_paged_select(None, None) == INVALID and kvx.kvx_paged_select_workspace_bytes(None) == 0
    assert _select(kvx, first=0, last=0) == _select(kvx, first=5, last=5) == _select(kvx, count=500) == _select(kvx, elem_dtype=_lib.KVX_KV_F16) == _lib.KVX_ERR_HIP
    assert _select(kvx, B=0, q=0, bounds=0, chosen=0, workspace=0) == _lib.KVX_OK
    for bad in (dict(num_pages=0), dict(Hkv=0), dict(B=-1), dict(Hq=0), dict(Hq=7), dict(max_pages=0), dict(count=0), dict(count=-1), dict(first=-1), dict(last=-1), dict(first=6, last=5),
                dict(first=2**31 - 1, last=2**31 - 1), dict(q=0), dict(q=4104), dict(q_stride_h=4), dict(bounds=0), dict(bounds=4100), dict(b_stride_page=-512), dict(b_stride_h=12),
                dict(block_table=0), dict(lens=0), dict(chosen=0), dict(bt_stride_b=-1)):
        assert _select(kvx, **bad) == INVALID, bad
    for bad in (dict(page_size=0), dict(page_size=8), dict(page_size=24), dict(page_size=2048), dict(D=96), dict(elem_dtype=_lib.KVX_KV_U8), dict(Hq=34), dict(Hkv=65536, Hq=65536),
                dict(B=65536), dict(max_pages=2**26), dict(B=60000, Hkv=1000, Hq=1000), dict(count=2**30 + 1), dict(count=2**31 - 1)):
        assert _select(kvx, **bad) == UNSUPPORTED, bad


@no_device
def test_decode_of_chosen_pages_is_checked(kvx):
    assert kvx.kvx_paged_decode_chosen(None, None, None) == INVALID and kvx.kvx_paged_decode_chosen_workspace_bytes(None, None) == 0
    a, _ = _decode_args()
    assert kvx.kvx_paged_decode_chosen(ctypes.byref(a), None, None) == INVALID
    assert _decode(kvx, chosen=dict(count=1)) == _decode(kvx, chosen=dict(count=2**31 - 1)) == _decode(kvx, chosen=dict(stride_b=0, stride_h=0)) == _lib.KVX_ERR_HIP
    assert _decode(kvx, B=0, q=0, chosen=dict(pages=0)) == _lib.KVX_OK
    for bad in (dict(pages=0), dict(count=0), dict(count=-5), dict(stride_b=-1), dict(stride_h=-1)):
        assert _decode(kvx, chosen=bad) == INVALID, bad
    for bad in (dict(B=-1), dict(Hq=7), dict(max_pages=0), dict(block_table=0), dict(lens=0), dict(q=0), dict(o=4104), dict(sm_scale=0.0), dict(sm_scale=math.nan)):
        assert _decode(kvx, **bad) == INVALID, bad
    for bad in (dict(Hq=34), dict(B=65536), dict(max_pages=2**26)):
        assert _decode(kvx, **bad) == UNSUPPORTED, bad


@no_device
def test_workspaces(kvx):
    """Checked before the launch."""
    for fields, chosen in ((dict(), dict()), (dict(B=500), dict(count=7)), (dict(Hq=32), dict(count=400))):
        need = kvx.kvx_paged_decode_chosen_workspace_bytes(*(ctypes.byref(x) for x in _decode_args((), chosen, **fields)))
        assert _decode(kvx, (), chosen, **fields, workspace_bytes=need) == _lib.KVX_ERR_HIP
        if need:
            assert _decode(kvx, (), chosen, **fields, workspace_bytes=need - 1) == _decode(kvx, (), chosen, **fields, workspace=4104) == _lib.KVX_ERR_WORKSPACE
    for fields in (dict(), dict(B=64, max_pages=8192), dict(count=5000)):
        need = kvx.kvx_paged_select_workspace_bytes(ctypes.byref(_select_args(**fields)))
        assert _select(kvx, **fields, workspace_bytes=need) == _lib.KVX_ERR_HIP
        if need:
            assert _select(kvx, **fields, workspace_bytes=need - 1) == _select(kvx, **fields, workspace=0) == _lib.KVX_ERR_WORKSPACE


def test_there_is_no_cpu_path():
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    pages, bounds = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 2, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, dtype=torch.int32)
    tables = rows.rope_tables(10, 64, 1e4, "cpu")
    for call in (lambda: paged_append(torch.zeros(4, 8 * 64, dtype=torch.bfloat16), 4, 2, 64, None, None, 0.0, *tables, lens, pages, pages, torch.zeros(4, dtype=torch.int64)),
                 lambda: paged_bounds(pages, bounds, table, lens), lambda: ops.paged_select(x, bounds, table, lens, 16, 2),
                 lambda: ops.paged_decode_chosen(x, pages, pages, table, lens, torch.zeros(4, 2, 1, dtype=torch.int32), 0.1)):
        with pytest.raises(RuntimeError, match="device"):
            call()


def test_a_pool_without_bounds_is_refused():
    pool = PagedKVCacheBuffers.__new__(PagedKVCacheBuffers)
    pool.k = pool.quant = pool.bounds = None
    for call in (lambda: pool.update_bounds(None, None), lambda: pool.select(None, None, None, 4)):
        with pytest.raises(ValueError, match="bounds=True"):
            call()
