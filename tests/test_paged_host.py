"""CPU: pools in 8 bits, rotation tables and the refusals of the cache
operators that need no device."""

from __future__ import annotations

import ctypes
import math
import os
import re
import shutil
import subprocess

import pytest
import torch

from imba_chess_b200 import _native, paged
from imba_chess_b200.kvpool import KVPool, KVSequence

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_native.LIB_PATH):
        from imba_chess_b200.build import build

        build()
    return _native.load()


def _pool(dtype=torch.float8_e4m3fn, dqk=64, dv=64, pages=8, device="cpu"):
    return KVPool(num_layers=2, num_heads=3, attention_dim=dqk, linear_dim=dv, num_pages=pages, dtype=dtype,
                  device=torch.device(device))


def test_pool_in_8_bits_layout():
    pool = _pool(dqk=32, dv=64)
    assert pool.data.dtype == torch.float8_e4m3fn and tuple(pool.data.shape) == (8, 2 * 3 * 16 * 96)
    assert pool.scales.dtype == torch.uint8 and tuple(pool.scales.shape) == (8, 2, 2, 3)
    assert pool.scales.data_ptr() == pool.data.data_ptr() + 8 * pool.page_elems  # behind the last page
    assert pool.page_bytes == pool.page_elems + 12
    cache = _native.CacheDesc(2, 3, 32, 64, _native.DTYPE_E4M3)
    assert _native.load().imba_cache_pool_bytes(ctypes.byref(cache), 8) == 8 * pool.page_bytes


@pytest.mark.parametrize("dqk,dv", [(16, 16), (48, 48), (64, 128), (128, 64), (96, 64), (256, 256), (64, 65)])
def test_pool_in_8_bits_refuses_other_head_sizes(lib, dqk, dv):
    with pytest.raises(ValueError, match="8 bits"):
        _pool(dqk=dqk, dv=dv)
    cache = _native.CacheDesc(1, 1, dqk, dv, _native.DTYPE_E4M3)
    assert lib.imba_cache_pool_bytes(ctypes.byref(cache), 1) == 0


def test_pages_start_afresh():
    pool = _pool()
    pool.scales.fill_(130)
    seq = KVSequence(pool)
    seq.reserve(33)
    pool.begin_pages()
    assert (pool.scales[seq.pages] == 0).all() and (pool.scales == 130).sum() == 5 * 12
    pool.scales.fill_(130)
    pool.begin_pages()  # nothing was handed out since
    assert (pool.scales == 130).all()
    seq.release()
    again = KVSequence(pool)
    again.reserve(1)
    pool.begin_pages()
    assert (pool.scales[again.pages] == 0).all()
    pool.begin_pages([7])
    assert (pool.scales[7] == 0).all()
    with pytest.raises(ValueError):
        pool.begin_pages([8])
    full = _pool(torch.float32)
    full.alloc(2)
    full.begin_pages()  # no scales: nothing to do
    assert full.scales is None and full._fresh == []


def test_rotary_turns():
    freq = [1.0, 10000 ** (-7 / 32), 1e-9, 0.0, -0.25, 9.5]
    rot = paged.Rotary(freq, device="cpu")
    for f, t in zip(freq, rot.turns.tolist()):
        for pos in (0, 1, 12345, 999_999):
            frac = (t * pos % 2**64) / 2**64
            want = math.fmod(f * pos, 2 * math.pi) / (2 * math.pi) % 1.0
            off = abs(frac - want)
            assert min(off, 1 - off) <= pos * abs(f) * 2**-52 + 2**-40, (f, pos)
    assert rot.rot_dim == 12 and rot.num_axes == 1 and rot.axis is None
    assert paged.Rotary([1.0, 2.0], device="cpu", axes=[0, 2]).num_axes == 3


@pytest.mark.parametrize("kw", [{"inv_freq": []}, {"inv_freq": [1.0] * 65}, {"inv_freq": [math.inf]},
                                {"inv_freq": [1.0], "layout": "neither"}, {"inv_freq": [1.0, 2.0], "axes": [0]},
                                {"inv_freq": [1.0], "axes": [8]}, {"inv_freq": [1.0], "axes": [-1]}])
def test_rotary_refusals(kw):
    with pytest.raises(ValueError):
        paged.Rotary(kw.pop("inv_freq"), device="cpu", **kw)


def test_cpu_pools_are_refused():
    with pytest.raises(ValueError, match="CUDA pool"):
        paged.AppendPlan(_pool(), [0])
    with pytest.raises(ValueError, match="CUDA pool"):
        paged.kv_read(_pool(torch.float32), 0, [0])


def test_library_refuses_malformed_calls(lib):
    """Every refusal comes before anything is launched, so no device is needed."""
    cache = _native.CacheDesc(2, 4, 64, 64, _native.DTYPE_E4M3)
    pool = _native.PoolDesc(1 << 20, 16)
    ok, arg, rng = _native.IMBA_OK, _native.IMBA_ERR_ARG, _native.IMBA_ERR_RANGE
    byref, big, at = ctypes.byref, 1 << 30, 1 << 20

    a = _native.AppendDesc(4, 0, _native.DTYPE_BF16, 0, at, at, at)

    def append(**kw):
        d = _native.AppendDesc.from_buffer_copy(a)
        c, p, plan, size = cache, pool, at, big
        for k, v in kw.items():
            if k in ("c", "p", "plan", "size"):
                c, p, plan, size = (v if k == "c" else c, v if k == "p" else p, v if k == "plan" else plan,
                                    v if k == "size" else size)
            elif k.startswith("rot_"):
                setattr(d.rotary, k[4:], v)
            else:
                setattr(d, k, v)
        return lib.imba_kv_append(None if c is None else byref(c), byref(p), byref(d), plan, size, None)

    assert append(num_rows=0) == ok
    assert append(c=None) == arg and append(num_rows=-1) == arg and append(k=None) == arg and append(v=None) == arg
    assert append(slots=None) == arg and append(src_dtype=2) == arg and append(plan=None) == arg
    assert append(layer=2) == rng and append(layer=-1) == rng
    assert append(size=64) == _native.IMBA_ERR_OOM and append(plan=at + 16) == arg
    assert append(p=_native.PoolDesc(None, 16)) == arg and append(p=_native.PoolDesc(at + 64, 16)) == arg
    assert append(p=_native.PoolDesc(at, 0)) == arg and append(p=_native.PoolDesc(at, 1 << 40)) == rng
    assert append(q=at) == arg and append(q=at, q_out=at) == arg  # no heads
    assert append(rot_rot_dim=3) == arg and append(rot_rot_dim=128) == arg and append(rot_rot_dim=64) == arg
    assert append(rot_rot_dim=64, rot_turns=at, rot_positions=at, rot_num_axes=9) == arg
    for bad in (_native.CacheDesc(0, 4, 64, 64, 2), _native.CacheDesc(2, 0, 64, 64, 2), _native.CacheDesc(2, 4, 64, 64, 3)):
        assert append(c=bad) == arg
    assert append(c=_native.CacheDesc(2, 4, 40, 40, 2)) == _native.IMBA_ERR_UNSUPPORTED
    assert append(c=_native.CacheDesc(2, 4, 160, 64, 0)) == _native.IMBA_ERR_UNSUPPORTED

    assert lib.imba_append_plan(byref(pool), 4, None, at, big, None, None) == arg
    assert lib.imba_append_plan(byref(pool), -1, at, at, big, None, None) == arg
    assert lib.imba_append_plan(byref(pool), 4, at, at, 64, None, None) == _native.IMBA_ERR_OOM
    assert lib.imba_append_plan_bytes(-1) == 0 and lib.imba_append_plan_bytes(1 << 30) == 0

    assert lib.imba_kv_read(byref(cache), byref(pool), 0, 0, None, 1, None, None, None, None) == ok
    assert lib.imba_kv_read(byref(cache), byref(pool), 5, 1, at, 1, at, at, None, None) == rng
    assert lib.imba_kv_read(byref(cache), byref(pool), 0, 1, at, 2, at, at, None, None) == arg
    assert lib.imba_kv_read(byref(cache), byref(pool), 0, 1, None, 1, at, at, None, None) == arg

    rows = _native.AttendDesc(4, 2, 2, 8, 0, 8)
    for name in ("seg_row_off", "row_vis", "group_page_off", "group_pages"):
        setattr(rows, name, at)
    args = _native.AttendArgs(0, _native.DTYPE_BF16, at, at)

    def attend(what="rows", c=cache, size=big, plan=at, **kw):
        r, g = _native.AttendDesc.from_buffer_copy(rows), _native.AttendArgs.from_buffer_copy(args)
        for k, v in kw.items():
            setattr(r if what == "rows" else g, k, v)
        return lib.imba_attend(byref(c), byref(pool), byref(r), byref(g), plan, size, None)

    assert attend(num_rows=0) == ok and attend(num_segs=0) == ok
    assert attend(num_rows=-1) == arg and attend(num_q_heads=6) == arg and attend(num_q_heads=0) == arg
    assert attend(num_segs=3) == arg  # a segment without a group
    assert attend(seg_row_off=None) == arg and attend(row_vis=None) == arg and attend(group_page_off=None) == arg
    assert attend(group_pages=None) == arg and attend(num_extra=1) == arg
    assert attend(num_group_pages=1 << 28) == rng and attend(num_rows=1 << 30) == _native.IMBA_ERR_UNSUPPORTED
    assert attend(size=256) == _native.IMBA_ERR_OOM and attend(plan=at + 4) == arg and attend(plan=None) == arg
    assert attend(c=_native.CacheDesc(2, 4, 64, 64, _native.DTYPE_BF16)) == _native.IMBA_ERR_UNSUPPORTED
    assert attend("args", layer=2) == rng and attend("args", dtype=2) == arg
    assert attend("args", q=None) == arg and attend("args", out=None) == arg
    assert attend("args", bias=at) == arg  # no positions
    assert lib.imba_attend_plan_bytes(byref(cache), byref(_native.AttendDesc(4, 2, 2, 8, 0, 6))) == 0


def test_library_refuses_sizes_past_32_bit_columns(lib):
    """Lists of more than 2^26 pages, and tables of more than 2^28 positions a side;
    pools whose slots are no int32."""
    byref = ctypes.byref
    cache, pool, at = _native.CacheDesc(2, 4, 64, 64, _native.DTYPE_E4M3), _native.PoolDesc(1 << 20, 4), 1 << 20
    most = (2**31 - 1) // 16
    assert lib.imba_cache_pool_bytes(byref(cache), most) == most * 2 * 4 * (16 * 128 + 2)
    assert lib.imba_cache_pool_bytes(byref(cache), most + 1) == 0 == lib.imba_cache_pool_bytes(byref(cache), 1 << 60)
    rows = _native.AttendDesc(4, 2, 2, 1 << 26, 0, 4)
    assert lib.imba_attend_plan_bytes(byref(cache), byref(rows)) > 0
    more = _native.AttendDesc(4, 2, 2, (1 << 26) + 1, 0, 4)
    assert lib.imba_attend_plan_bytes(byref(cache), byref(more)) == 0
    for name in ("seg_row_off", "row_vis", "group_page_off", "group_pages", "positions"):
        setattr(rows, name, at)
    args = _native.AttendArgs(layer=0, dtype=_native.DTYPE_BF16, q=at, out=at, scale=1.0, max_pos=(1 << 28) + 1, bias=at)
    assert lib.imba_attend(byref(cache), byref(pool), byref(rows), byref(args), at, 1 << 40, None) == _native.IMBA_ERR_UNSUPPORTED


def test_cache_struct_layouts_match_c(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host C++ compiler")
    text = open(os.path.join(ROOT, "include", "imba_b200.h")).read()
    want, lines = [], []
    for c, py in (("imba_cache_desc", _native.CacheDesc), ("imba_rotary_desc", _native.RotaryDesc),
                  ("imba_append_desc", _native.AppendDesc), ("imba_attend_desc", _native.AttendDesc),
                  ("imba_attend_args", _native.AttendArgs)):
        assert re.search(rf"\b{c};", text)
        lines.append(f"sizeof({c})")
        want.append(ctypes.sizeof(py))
        for name, _ in py._fields_:
            lines.append(f"offsetof({c}, {name})")
            want.append(getattr(py, name).offset)
    src = tmp_path / "sizes.cc"
    src.write_text('#include <cstdio>\n#include <cstddef>\n#include "imba_b200.h"\nint main(){'
                   + "".join(f'printf("%zu ", (size_t)({x}));' for x in lines) + "}\n")
    exe = tmp_path / "sizes"
    subprocess.run([gxx, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want
