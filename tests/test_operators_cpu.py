"""The C entries of the backward pass and of the 4-bit cache refuse bad arguments before any launch, and their
argument blocks match the header (no GPU needed)."""
from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

import flash_atten
import hip_lib
import kv4

HEADER = Path(__file__).resolve().parent.parent / "include" / "fa_gfx950.h"


def test_struct_layouts_match_the_header(tmp_path):
    structs = {"fa_bwd_args": hip_lib.FaBwdArgs, "kv4_cache": hip_lib.Kv4CacheArgs,
               "kv4_append_args": hip_lib.Kv4AppendArgs, "kv4_attend_args": hip_lib.Kv4AttendArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    out = dict(x.rsplit(" ", 1) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for cname, cls in structs.items():
        assert int(out[cname]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(out[f"{cname}.{f}"]) == getattr(cls, f).offset, f"{cname}.{f}"


def _i64(*x):
    return (ctypes.c_int64 * len(x))(*x)


def _bwd(**over):
    a = hip_lib.FaBwdArgs()
    for name in ("q", "k", "v", "o", "dout", "lse", "dq", "dk", "dv", "workspace"):
        setattr(a, name, 256)  # never dereferenced: every case below fails validation first
    for name in ("q", "k", "v", "o", "dout", "dq", "dk", "dv"):
        setattr(a, name + "_stride", _i64(8192, 4096, 64, 1))
    a.lse_stride = _i64(128, 64, 1)
    a.B, a.H, a.H_kv, a.M, a.N, a.D = 1, 2, 2, 64, 64, 64
    a.sm_scale, a.dtype, a.workspace_bytes = 0.125, 0, 1 << 30
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code,needle", [
    ({"D": 96}, hip_lib.FA_ENOTSUP, "head dim"), ({"dtype": 2}, hip_lib.FA_ENOTSUP, "dtype"),
    ({"H": 3}, hip_lib.FA_EINVAL, "multiple of kv heads"), ({"M": -1}, hip_lib.FA_EINVAL, "invalid sizes"),
    ({"sm_scale": 0.0}, hip_lib.FA_EINVAL, "sm_scale"), ({"sm_scale": float("inf")}, hip_lib.FA_EINVAL, "sm_scale"),
    ({"sm_scale": 3e38}, hip_lib.FA_EINVAL, "sm_scale"),
    ({"q": None}, hip_lib.FA_EINVAL, "null q"), ({"dv": None}, hip_lib.FA_EINVAL, "null dv"),
    ({"lse": None}, hip_lib.FA_EINVAL, "null lse"), ({"k": 264}, hip_lib.FA_EINVAL, "k must be 16-byte aligned"),
    ({"v_stride": _i64(8192, 4096, 64, 2)}, hip_lib.FA_EINVAL, "head-dim stride of v"),
    ({"o_stride": _i64(8192, 4092, 64, 1)}, hip_lib.FA_EINVAL, "strides of o"),
    ({"dout_stride": _i64(8192, 4096, 0, 1)}, hip_lib.FA_EINVAL, "row stride 0 of dout"),
    ({"k_stride": _i64(8192, 4096, 1 << 23, 1)}, hip_lib.FA_EINVAL, "row stride"),
    ({"workspace": None}, hip_lib.FA_EWORKSPACE, "workspace of"), ({"workspace_bytes": 64}, hip_lib.FA_EWORKSPACE, "got 64"),
    ({"workspace": 272}, hip_lib.FA_EINVAL, "256-byte aligned"),
])
def test_backward_refusals(over, code, needle):
    assert hip_lib.load().fa_bwd(ctypes.byref(_bwd(**over)), None) == code
    assert needle in hip_lib.last_error()


def test_empty_calls_do_nothing():
    lib = hip_lib.load()
    assert lib.fa_bwd(ctypes.byref(_bwd(B=0)), None) == hip_lib.FA_OK
    assert lib.fa_bwd(ctypes.byref(_bwd(M=0, N=0)), None) == hip_lib.FA_OK
    assert lib.fa_bwd(None, None) == lib.kv4_append(None, None) == lib.kv4_attend(None, None) == hip_lib.FA_EINVAL
    assert lib.kv4_append(ctypes.byref(_append(rows=0)), None) == hip_lib.FA_OK
    assert lib.kv4_attend(ctypes.byref(_attend(M=0)), None) == hip_lib.FA_OK
    assert lib.fa_bwd_workspace_bytes(0, 1, 1, 1, 1, 64, 0) == lib.kv4_attend_workspace_bytes(1, 1, 1, 64, 1) == 0
    assert lib.kv4_attend_workspace_bytes(2, 4, 3, 64, 5) == 5 * 24 * (64 * 4 + 8)


def _cache(**over):
    c = hip_lib.Kv4CacheArgs()
    c.k_codes = c.k_scales = c.v_codes = c.v_scales = 256
    c.code_stride, c.scale_stride = _i64(4096, 2048), _i64(256, 128)
    c.B, c.H_kv, c.D, c.dtype, c.rows, c.capacity = 1, 2, 64, 1, 64, 50
    for k, v in over.items():
        setattr(c, k, v)
    return c


def _append(cache=None, **over):
    a = hip_lib.Kv4AppendArgs()
    a.cache = cache or _cache()
    a.k = a.v = a.start = 256
    a.k_stride = a.v_stride = a.k_values_stride = a.v_values_stride = _i64(1024, 512, 64, 1)
    a.rows = 8
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _attend(cache=None, **over):
    a = hip_lib.Kv4AttendArgs()
    a.cache = cache or _cache()
    a.q = a.o = a.start = 256
    a.q_stride = a.o_stride = _i64(1024, 512, 64, 1)
    a.H, a.M, a.sm_scale, a.causal, a.splits = 4, 2, 0.125, 1, 1
    for k, v in over.items():
        setattr(a, k, v)
    return a


CACHE_REFUSALS = [
    ({"D": 32}, hip_lib.FA_ENOTSUP, "head dim"), ({"dtype": 5}, hip_lib.FA_ENOTSUP, "dtype"),
    ({"H_kv": 0}, hip_lib.FA_EINVAL, "invalid cache sizes"), ({"rows": 50}, hip_lib.FA_EINVAL, "multiple of 32"),
    ({"capacity": 65}, hip_lib.FA_EINVAL, "at least the capacity"),
    ({"capacity": (1 << 30) + 1, "rows": (1 << 30) + 32}, hip_lib.FA_ENOTSUP, "is beyond"), ({"v_scales": None}, hip_lib.FA_EINVAL, "null cache"),
    ({"k_codes": 264}, hip_lib.FA_EINVAL, "16-byte aligned"), ({"code_stride": _i64(4096, 2040)}, hip_lib.FA_EINVAL, "multiples of 16"),
]


@pytest.mark.parametrize("over,code,needle", CACHE_REFUSALS)
def test_cache_refusals(over, code, needle):
    lib = hip_lib.load()
    assert lib.kv4_append(ctypes.byref(_append(_cache(**over))), None) == code
    assert needle in hip_lib.last_error()
    assert lib.kv4_attend(ctypes.byref(_attend(_cache(**over))), None) == code
    assert needle in hip_lib.last_error()


@pytest.mark.parametrize("over,code,needle", [
    ({"rows": -1}, hip_lib.FA_EINVAL, "row count"), ({"k": None}, hip_lib.FA_EINVAL, "null k"),
    ({"v": 258}, hip_lib.FA_EINVAL, "16-byte aligned"), ({"start": None}, hip_lib.FA_EINVAL, "null start"),
    ({"k_values": 256}, hip_lib.FA_EINVAL, "go together"), ({"k_stride": _i64(1024, 512, 32, 1)}, hip_lib.FA_EINVAL, "row stride 32 of k"),
])
def test_append_refusals(over, code, needle):
    assert hip_lib.load().kv4_append(ctypes.byref(_append(**over)), None) == code
    assert needle in hip_lib.last_error()


@pytest.mark.parametrize("over,code,needle", [
    ({"H": 3}, hip_lib.FA_EINVAL, "multiple of kv heads"), ({"M": -1}, hip_lib.FA_EINVAL, "invalid sizes"),
    ({"sm_scale": float("nan")}, hip_lib.FA_EINVAL, "sm_scale"), ({"splits": 0}, hip_lib.FA_EINVAL, "splits"),
    ({"splits": 4097}, hip_lib.FA_EINVAL, "splits"), ({"q": None}, hip_lib.FA_EINVAL, "null q"),
    ({"o": 260}, hip_lib.FA_EINVAL, "o must be 8-byte aligned"), ({"start": None}, hip_lib.FA_EINVAL, "null start"),
    ({"splits": 2}, hip_lib.FA_EWORKSPACE, "split workspace"), ({"M": 1 << 30, "H": 8}, hip_lib.FA_EINVAL, "too many query rows"),
])
def test_attend_refusals(over, code, needle):
    assert hip_lib.load().kv4_attend(ctypes.byref(_attend(**over)), None) == code
    assert needle in hip_lib.last_error()


def test_python_refusals_without_a_gpu():
    x = torch.zeros(1, 2, 4, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU tensor"):
        flash_atten.attention_backward(x, x, x, x, x, torch.zeros(1, 2, 4))
    with pytest.raises(ValueError, match="lives on a GPU"):
        kv4.Kv4Cache(1, 1, 8, 64, dtype=torch.float16, device="cpu")
    with pytest.raises(hip_lib.FaUnsupportedError):
        kv4.Kv4Cache(1, 1, 8, 96, dtype=torch.float16)
    with pytest.raises(hip_lib.FaUnsupportedError):
        kv4.Kv4Cache(1, 1, 8, 64, dtype=torch.float32)
    with pytest.raises(hip_lib.FaUnsupportedError, match="is beyond"):
        kv4.Kv4Cache(1, 1, (1 << 30) + 1, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="invalid cache sizes"):
        kv4.Kv4Cache(1, 1, 0, 64, dtype=torch.float16)


def test_splits_rule():
    """Grids that fill the chip are not split; no split has less than 256 keys of a full cache."""
    assert kv4.choose_splits(64, 32, 8, 1, 128, 65536) == 1
    assert kv4.choose_splits(1, 32, 8, 1, 128, 255) == 1
    for B, H, Hk, M, D, cap in ((1, 32, 8, 1, 128, 8192), (1, 12, 2, 4, 128, 100000), (2, 28, 4, 509, 128, 16384), (1, 1, 1, 1, 64, 1 << 20)):
        n = kv4.choose_splits(B, H, Hk, M, D, cap)
        assert 1 <= n <= max(1, cap // 256) and n <= 4096
