"""CPU-side checks of the paged cache's boundary: argument layouts, what the entry points refuse (with made-up pointers: nothing is launched), what the
Python functions refuse, and the angles of long contexts."""
import ctypes
import math
import os
import subprocess
from types import SimpleNamespace

import pytest
import torch

from keys_values_amd import _lib
from keys_values_amd.attention import ops
from keys_values_amd.kvcache.paged import PagedKVCacheBuffers, paged_read, paged_write
from keys_values_amd.longctx import ops as rows

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "kvx.h")
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up: where nothing can be launched")


def test_struct_layouts_match_c(tmp_path):
    structs = {"kvx_rotary_args": _lib.RotaryArgs, "kvx_pages": _lib.Pages, "kvx_paged_write_args": _lib.PagedWriteArgs, "kvx_paged_read_args": _lib.PagedReadArgs,
               "kvx_paged_decode_args": _lib.PagedDecodeArgs}
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


def _pages(p, **fields):
    p.num_pages, p.page_size, p.Hkv, p.D, p.kv_dtype = 100, 16, 2, 128, _lib.KVX_KV_BF16
    p.k = p.v = p.k_scale = p.k_zp = p.v_scale = p.v_zp = 4096
    p.k_stride_t = p.v_stride_t = 128
    p.k_stride_h = p.v_stride_h = 16 * 128
    p.k_stride_page = p.v_stride_page = 2 * 16 * 128
    p.qs_stride_h, p.qs_stride_page = 16, 32
    for name, value in fields.items():
        setattr(p, name, value)


def _write(kvx, pages=(), **fields):
    a = _lib.PagedWriteArgs()
    _pages(a.pages, **dict(pages))
    a.tokens, a.key, a.value, a.slots = 5, 4096, 4096, 4096
    a.key_stride_t = a.value_stride_t = 256
    a.key_stride_h = a.value_stride_h = 128
    for name, value in fields.items():
        setattr(a, name, value)
    return kvx.kvx_paged_write(ctypes.byref(a), None)


def _read(kvx, pages=(), **fields):
    a = _lib.PagedReadArgs()
    _pages(a.pages, **dict(pages))
    a.B, a.length, a.max_pages, a.block_table, a.lens, a.bt_stride_b, a.key, a.value = 3, 50, 7, 4096, 4096, 7, 4096, 4096
    a.key_stride_b = a.value_stride_b = 2 * 50 * 128
    a.key_stride_h = a.value_stride_h = 50 * 128
    a.key_stride_t = a.value_stride_t = 128
    for name, value in fields.items():
        setattr(a, name, value)
    return kvx.kvx_paged_read(ctypes.byref(a), None)


def _decode_args(pages=(), **fields):
    a = _lib.PagedDecodeArgs()
    _pages(a.pages, **dict(pages))
    a.B, a.Hq, a.max_pages, a.sm_scale, a.q, a.block_table, a.lens, a.o, a.bt_stride_b = 3, 8, 7, 0.1, 4096, 4096, 4096, 4096, 7
    a.q_stride_b = a.o_stride_b = 8 * 128
    a.q_stride_h = a.o_stride_h = 128
    a.workspace, a.workspace_bytes = 4096, 2**40
    for name, value in fields.items():
        setattr(a, name, value)
    return a


def _decode(kvx, pages=(), **fields):
    return kvx.kvx_paged_decode(ctypes.byref(_decode_args(pages, **fields)), None)


BAD_PAGES = [
    (dict(num_pages=0), "INVALID"), (dict(Hkv=0), "INVALID"), (dict(k=0), "INVALID"), (dict(v=4100), "INVALID"), (dict(k_stride_t=132), "INVALID"),
    (dict(v_stride_page=-4096), "INVALID"), (dict(page_size=0), "UNSUPPORTED"), (dict(page_size=8), "UNSUPPORTED"), (dict(page_size=48), "UNSUPPORTED"),
    (dict(page_size=2048), "UNSUPPORTED"), (dict(D=96), "UNSUPPORTED"), (dict(kv_dtype=6), "UNSUPPORTED"), (dict(kv_dtype=-1), "UNSUPPORTED"),
    (dict(k_stride_t=64), "UNSUPPORTED"), (dict(v_stride_t=2**20), "UNSUPPORTED"), (dict(Hkv=65536), "UNSUPPORTED"),
    (dict(k_stride_page=2**31), "UNSUPPORTED"), (dict(v_stride_page=2**40), "UNSUPPORTED"), (dict(k_stride_h=2**31), "UNSUPPORTED"), (dict(kv_dtype=_lib.KVX_KV_U8, qs_stride_page=2**30), "UNSUPPORTED"),
    (dict(kv_dtype=_lib.KVX_KV_U8, k_scale=0), "INVALID"), (dict(kv_dtype=_lib.KVX_KV_U8, v_zp=4100), "INVALID"),
    (dict(kv_dtype=_lib.KVX_KV_U8, qs_stride_h=18), "INVALID"), (dict(kv_dtype=_lib.KVX_KV_U8, k_stride_t=136), "INVALID"),
]


@no_device
@pytest.mark.parametrize("call", [_write, _read, _decode])
def test_pages_are_checked(kvx, call):
    for good in ({}, dict(kv_dtype=_lib.KVX_KV_U8), dict(kv_dtype=_lib.KVX_KV_U4_F16, k_stride_t=64, v_stride_t=64), dict(page_size=1024), dict(D=64), dict(k_scale=0)):
        assert call(kvx, good) == _lib.KVX_ERR_HIP, good  # no device
    for bad, status in BAD_PAGES:
        assert call(kvx, bad) == getattr(_lib, "KVX_ERR_" + status), bad
        assert kvx.kvx_last_error()


@no_device
def test_write_is_checked(kvx):
    invalid, unsupported = _lib.KVX_ERR_INVALID, _lib.KVX_ERR_UNSUPPORTED
    assert kvx.kvx_paged_write(None, None) == invalid
    assert _write(kvx, tokens=0, key=0, value=0, slots=0) == _lib.KVX_OK
    for bad in (dict(tokens=-1), dict(key=0), dict(value=0), dict(slots=0), dict(key=4104), dict(value_stride_t=260), dict(key_stride_h=4)):
        assert _write(kvx, **bad) == invalid, bad
    assert _write(kvx, tokens=2**31) == _write(kvx, tokens=2**30) == unsupported


@no_device
def test_read_is_checked(kvx):
    invalid, unsupported = _lib.KVX_ERR_INVALID, _lib.KVX_ERR_UNSUPPORTED
    assert kvx.kvx_paged_read(None, None) == invalid
    assert _read(kvx, B=0) == _read(kvx, length=0, key=0, value=0) == _lib.KVX_OK
    for bad in (dict(B=-1), dict(length=-1), dict(max_pages=0), dict(block_table=0), dict(lens=0), dict(key=0), dict(value=4104), dict(key_stride_t=130), dict(bt_stride_b=-1)):
        assert _read(kvx, **bad) == invalid, bad
    for bad in (dict(B=65536), dict(length=2**30), dict(max_pages=2**26), dict(B=60000, length=2**20)):
        assert _read(kvx, **bad) == unsupported, bad


@no_device
def test_decode_is_checked(kvx):
    invalid, unsupported = _lib.KVX_ERR_INVALID, _lib.KVX_ERR_UNSUPPORTED
    assert kvx.kvx_paged_decode(None, None) == invalid and kvx.kvx_paged_decode_workspace_bytes(None) == 0
    assert _decode(kvx, B=0, q=0, o=0, workspace=0) == _lib.KVX_OK
    for bad in (dict(B=-1), dict(Hq=0), dict(Hq=7), dict(max_pages=0), dict(block_table=0), dict(lens=0), dict(q=0), dict(o=4104), dict(q_stride_h=12), dict(sm_scale=0.0),
                dict(sm_scale=-1.0), dict(sm_scale=math.nan), dict(bt_stride_b=-1)):
        assert _decode(kvx, **bad) == invalid, bad
    for bad in (dict(Hq=34), dict(B=65536), dict(max_pages=2**26), dict(B=60000, max_pages=2**20)):
        assert _decode(kvx, **bad) == unsupported, bad


@no_device
def test_workspace_of_decode(kvx):
    """Checked before the launch; none where no sequence is split."""
    for fields in (dict(), dict(max_pages=2000), dict(B=500, max_pages=4000), dict(Hq=32, max_pages=300)):
        a = _decode_args(**fields)
        need = kvx.kvx_paged_decode_workspace_bytes(ctypes.byref(a))
        assert _decode(kvx, **fields, workspace_bytes=need) == _lib.KVX_ERR_HIP
        if need:
            assert _decode(kvx, **fields, workspace_bytes=need - 1) == _decode(kvx, **fields, workspace=0) == _decode(kvx, **fields, workspace=4104) == _lib.KVX_ERR_WORKSPACE
    assert kvx.kvx_paged_decode_workspace_bytes(ctypes.byref(_decode_args(Hq=7))) == 0


def _rotary(kvx, **fields):
    a = _lib.RotaryArgs()
    a.qkv, a.stride_t, a.tokens, a.Hq, a.Hkv, a.D, a.rotary_dim, a.elem_dtype, a.table_rows = 4096, 12 * 128, 9, 8, 2, 128, 64, _lib.KVX_KV_BF16, 50
    a.cos = a.sin = a.positions = a.q_weight = a.k_weight = 4096
    for name, value in fields.items():
        setattr(a, name, value)
    return kvx.kvx_rotary(ctypes.byref(a), None)


@no_device
def test_rotary_is_checked(kvx):
    assert kvx.kvx_rotary(None, None) == _lib.KVX_ERR_INVALID
    assert _rotary(kvx) == _rotary(kvx, q_weight=0, k_weight=0) == _rotary(kvx, tokens=1, stride_t=0) == _rotary(kvx, rotary_dim=128, interleaved=1) == _lib.KVX_ERR_HIP
    assert _rotary(kvx, tokens=0, qkv=0) == _lib.KVX_OK
    for bad in (dict(tokens=-1), dict(Hq=0), dict(Hkv=0), dict(qkv=0), dict(cos=0), dict(sin=4100), dict(positions=0), dict(q_weight=0), dict(k_weight=4100),
                dict(stride_t=1279), dict(stride_t=1284), dict(qkv=4104), dict(table_rows=0)):
        assert _rotary(kvx, **bad) == _lib.KVX_ERR_INVALID, bad
    for bad in (dict(D=96), dict(rotary_dim=0), dict(rotary_dim=8), dict(rotary_dim=144), dict(rotary_dim=-16), dict(elem_dtype=_lib.KVX_KV_U8), dict(Hq=65536),
                dict(tokens=2**31)):
        assert _rotary(kvx, **bad) == _lib.KVX_ERR_UNSUPPORTED, bad


def test_there_is_no_cpu_path():
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    pages = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, dtype=torch.int32)
    tables = rows.rope_tables(10, 64, 1e4, "cpu")
    for call in (lambda: paged_write(x, x, pages, pages, torch.zeros(4, dtype=torch.int64)), lambda: paged_read(pages, pages, table, lens, 5),
                 lambda: ops.paged_decode(x, pages, pages, table, lens, 0.1), lambda: PagedKVCacheBuffers(2, 16, 2, 64, device="cpu"),
                 lambda: rows.rotary_(torch.zeros(4, 8 * 64, dtype=torch.bfloat16), 4, 2, 64, None, None, 0.0, *tables, lens)):
        with pytest.raises(RuntimeError, match="device"):
            call()


@pytest.mark.parametrize("error,kwargs", [
    (ValueError, dict(num_pages=0)), (ValueError, dict(page_size=24)), (ValueError, dict(page_size=8)), (ValueError, dict(n_query_groups=0)), (ValueError, dict(num_bits=2)),
    (NotImplementedError, dict(head_size=80)), (NotImplementedError, dict(dtype=torch.float32)),
])
def test_pools_are_checked(error, kwargs):
    with pytest.raises(error):
        PagedKVCacheBuffers(**{**dict(num_pages=4, page_size=16, n_query_groups=2, head_size=64, device="cpu"), **kwargs})
    with pytest.raises(ValueError, match="head_size and dtype"):
        paged_read(None, None, None, None, 4, quant=())


def test_slots_are_checked():
    slots, pool = PagedKVCacheBuffers.slots, SimpleNamespace(page_size=16)
    table = torch.tensor([[3, 1], [0, -1]], dtype=torch.int32)
    assert slots(pool, table, torch.tensor([[0, 17], [-1, 16]])).tolist() == [48, 17, -1, -1]
    assert slots(pool, table[:0], torch.empty(0, 5, dtype=torch.int32)).shape == (0,)
    for bad, positions in ((table[:, :0], torch.zeros(2, 1)), (table[0], torch.zeros(2, 1)), (table, torch.zeros(1, 4)), (table, torch.zeros(3, 4)), (table, torch.zeros(2))):
        with pytest.raises(ValueError):
            slots(pool, bad, positions.int())


def test_a_context_without_a_turn_is_refused():
    rows.RopeScaling("yarn", 2.0, original_context=7)
    rows.RopeScaling("linear", 2.0, original_context=1)
    for kwargs in (dict(original_context=6), dict(original_context=60, beta_slow=10.0)):
        with pytest.raises(ValueError):
            rows.RopeScaling("yarn", 2.0, **kwargs)


# ---- angles of long contexts ----------------------------------------------------------------------------------------


def _half_step(x):
    return 2.0**-24 * abs(x) + 2.0**-149


def test_tables_without_scaling_are_as_before():
    inv = 1.0 / (1e6 ** (torch.arange(0, 128, 2, dtype=torch.float32) / 128))
    angle = torch.arange(300, dtype=torch.float32).unsqueeze(-1) * inv
    cos, sin = rows.rope_tables(300, 128, 1e6, "cpu")
    assert torch.equal(cos, angle.cos()) and torch.equal(sin, angle.sin())


@pytest.mark.parametrize("n", [16, 64, 128])
def test_tables_of_a_part_are_exact(n):
    cos, sin = rows.rope_tables(131073, 128, 1e4, "cpu", rotary_dim=n)
    assert cos.shape == sin.shape == (131073, n // 2) and cos.dtype == torch.float32
    for p in (0, 1, 4095, 131072):
        for j in range(0, n // 2, 5):
            a = p * 1e4 ** (-2 * j / n)
            # an angle in 64 bits is off by p 2^-50 at most
            assert abs(cos[p, j].item() - math.cos(a)) <= _half_step(math.cos(a)) + p * 2.0**-50
            assert abs(sin[p, j].item() - math.sin(a)) <= _half_step(math.sin(a)) + p * 2.0**-50


def _frequency(s, j, n, base):
    """Pair j's angle per position, straight from the definitions."""
    f = base ** (-2 * j / n)
    if s.kind == "linear":
        return f / s.factor
    if s.kind == "ntk":
        return (base * s.factor ** (n / (n - 2))) ** (-2 * j / n)
    if s.kind == "banded":
        wave = 2 * math.pi / f
        if wave < s.original_context / s.high_freq_factor:
            return f
        if wave > s.original_context / s.low_freq_factor:
            return f / s.factor
        keep = (s.original_context / wave - s.low_freq_factor) / (s.high_freq_factor - s.low_freq_factor)
        return (1 - keep) * f / s.factor + keep * f
    where = [n * math.log(s.original_context / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (s.beta_fast, s.beta_slow)]
    low, high = max(math.floor(where[0]), 0), min(math.ceil(where[1]), n - 1)
    ramp = min(max((j - low) / (high - low), 0.0), 1.0)
    return f / s.factor * ramp + f * (1 - ramp)


@pytest.mark.parametrize("scaling", [
    rows.RopeScaling("linear", 4.0), rows.RopeScaling("ntk", 8.0), rows.RopeScaling("banded", 8.0, 8192), rows.RopeScaling("banded", 32.0, 4096, 2.0, 5.0),
    rows.RopeScaling("yarn", 4.0, 32768), rows.RopeScaling("yarn", 16.0, 4096, attention_factor=1.0), rows.RopeScaling("linear", 1.0),
])
@pytest.mark.parametrize("base,n", [(1e4, 64), (1e6, 128)])
def test_angles_for_long_contexts(scaling, base, n):
    got = scaling.frequencies(n, base)
    assert got.dtype == torch.float64 and got.shape == (n // 2,)
    for j in range(n // 2):
        want = _frequency(scaling, j, n, base)
        assert abs(got[j].item() - want) <= 1e-12 * want
    m = 1.0 if scaling.kind != "yarn" else scaling.attention_factor or 0.1 * math.log(scaling.factor) + 1.0
    cos, sin = rows.rope_tables(5000, n, base, "cpu", scaling=scaling)
    for p in (0, 7, 4999):
        a = p * _frequency(scaling, 3, n, base)
        assert abs(cos[p, 3].item() - m * math.cos(a)) <= _half_step(2.0) + 1e-11 and abs(sin[p, 3].item() - m * math.sin(a)) <= _half_step(2.0) + 1e-11


@pytest.mark.parametrize("kwargs", [
    dict(kind="dynamic", factor=2.0), dict(kind="linear", factor=0.5), dict(kind="linear", factor=math.nan), dict(kind="yarn", factor=2.0, original_context=0),
    dict(kind="banded", factor=2.0, low_freq_factor=4.0), dict(kind="yarn", factor=2.0, beta_slow=40.0),
])
def test_scalings_are_checked(kwargs):
    with pytest.raises(ValueError):
        rows.RopeScaling(**kwargs)
    for n in (0, 7, 130):
        with pytest.raises(ValueError):
            rows.rope_tables(10, 128, 1e4, "cpu", rotary_dim=n)
