"""The C entries of the paged 8-bit cache refuse bad arguments before any launch, their argument blocks match the header,
their sources honour NaN, and the tests' model follows the format's definition (no GPU needed)."""
from __future__ import annotations

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

import build_lib
import hip_lib
import kv8
import kv8_model
import flash_atten

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "fa_gfx950.h"
PAGED = sorted((Path(build_lib.__file__).resolve().parent / "csrc" / "paged").glob("*.hip"))


def test_struct_layouts_match_the_header(tmp_path):
    structs = {"kv8_cache": hip_lib.Kv8CacheArgs, "kv8_append_args": hip_lib.Kv8AppendArgs,
               "kv8_attend_args": hip_lib.Kv8AttendArgs, "kv8_reserve_args": hip_lib.Kv8ReserveArgs,
               "kv8_compact_args": hip_lib.Kv8CompactArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    lines += ['  printf("fork %d\\n", KV8_MAX_FORK);', '  printf("capacity %d\\n", KV8_MAX_CAPACITY);']
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    out = dict(x.rsplit(" ", 1) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for cname, cls in structs.items():
        assert int(out[cname]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(out[f"{cname}.{f}"]) == getattr(cls, f).offset, f"{cname}.{f}"
    assert int(out["fork"]) == kv8.MAX_FORK and int(out["capacity"]) == kv8.MAX_CAPACITY


@pytest.mark.parametrize("path", PAGED, ids=lambda p: p.name)
def test_sources_honour_nan_and_keep_packed_fp32_off(path):
    flags = build_lib.flags_for(path)
    assert not any("honor-nan" in f or f in ("-ffast-math", "-ffinite-math-only", "-mno-amdgpu-ieee") for f in flags)
    assert "-packed-fp32-ops" in flags and flags[flags.index("-packed-fp32-ops") - 1] == "-Xclang"


def test_the_build_takes_the_folder():
    assert len(PAGED) == 3
    assert any("kv8_attend_kernel" in name for name in hip_lib.compiled_resources())


def _i64(*x):
    return (ctypes.c_int64 * len(x))(*x)


def _cache(**over):
    c = hip_lib.Kv8CacheArgs()
    c.data = c.table = c.refs = 256  # never dereferenced: every case below fails validation first
    c.B, c.H_kv, c.D, c.dtype, c.page, c.pages, c.columns, c.capacity, c.layers = 1, 2, 64, 1, 64, 8, 4, 250, 1
    c.page_stride, c.layer_stride = 16512, 16512 * 8
    for k, v in over.items():
        setattr(c, k, v)
    return c


def _append(cache=None, **over):
    a = hip_lib.Kv8AppendArgs()
    a.cache = cache or _cache()
    a.k = a.v = a.start = 256
    a.k_stride = a.v_stride = a.k_values_stride = a.v_values_stride = _i64(1024, 512, 64, 1)
    a.rows = 8
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _attend(cache=None, **over):
    a = hip_lib.Kv8AttendArgs()
    a.cache = cache or _cache()
    a.q = a.o = a.start = 256
    a.q_stride = a.o_stride = _i64(1024, 512, 64, 1)
    a.H, a.M, a.sm_scale, a.causal, a.splits = 4, 2, 0.125, 1, 1
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _reserve(cache=None, **over):
    a = hip_lib.Kv8ReserveArgs()
    a.cache = cache or _cache()
    a.start = a.missing = a.workspace = 256
    a.workspace_bytes, a.rows = 1 << 30, 5
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _compact(cache=None, **over):
    a = hip_lib.Kv8CompactArgs()
    a.cache = cache or _cache()
    a.used = a.workspace = 256
    a.workspace_bytes = 1 << 30
    for k, v in over.items():
        setattr(a, k, v)
    return a


CACHE_REFUSALS = [
    ({"D": 32}, hip_lib.FA_ENOTSUP, "head dim"), ({"dtype": 5}, hip_lib.FA_ENOTSUP, "dtype"),
    ({"H_kv": 0}, hip_lib.FA_EINVAL, "invalid cache sizes"), ({"layers": 0}, hip_lib.FA_EINVAL, "invalid cache sizes"),
    ({"pages": 0}, hip_lib.FA_EINVAL, "invalid cache sizes"), ({"B": -1}, hip_lib.FA_EINVAL, "invalid cache sizes"),
    ({"page": 48}, hip_lib.FA_ENOTSUP, "pages of 48"), ({"capacity": 257}, hip_lib.FA_EINVAL, "do not hold"),
    ({"capacity": (1 << 30) + 1, "columns": 1 << 28}, hip_lib.FA_ENOTSUP, "is beyond"),
    ({"pages": (1 << 30) + 1}, hip_lib.FA_ENOTSUP, "pages are beyond"), ({"H_kv": (1 << 20) + 1}, hip_lib.FA_ENOTSUP, "beyond 2^20"),
    ({"B": 1 << 20, "columns": 1 << 11}, hip_lib.FA_EINVAL, "page table too large"),
    ({"table": None}, hip_lib.FA_EINVAL, "null cache"), ({"refs": None}, hip_lib.FA_EINVAL, "null cache"),
    ({"data": None}, hip_lib.FA_EINVAL, "null cache"), ({"data": 264}, hip_lib.FA_EINVAL, "16-byte aligned"),
    ({"page_stride": 16520}, hip_lib.FA_EINVAL, "16-byte aligned"), ({"page_stride": 16384}, hip_lib.FA_EINVAL, "is under a page"),
]


@pytest.mark.parametrize("over,code,needle", CACHE_REFUSALS)
def test_cache_refusals(over, code, needle):
    lib = hip_lib.load()
    c = _cache(**over)
    for call in (lambda: lib.kv8_append(ctypes.byref(_append(c)), None), lambda: lib.kv8_attend(ctypes.byref(_attend(c)), None),
                 lambda: lib.kv8_reserve(ctypes.byref(_reserve(c)), None), lambda: lib.kv8_compact(ctypes.byref(_compact(c)), None),
                 lambda: lib.kv8_fork(ctypes.byref(c), 256, None), lambda: lib.kv8_truncate(ctypes.byref(c), 256, None)):
        assert call() == code
        assert needle in hip_lib.last_error()
    assert lib.kv8_reserve_workspace_bytes(ctypes.byref(c), 4) == lib.kv8_compact_workspace_bytes(ctypes.byref(c)) == 0


@pytest.mark.parametrize("over,code,needle", [
    ({"rows": -1}, hip_lib.FA_EINVAL, "row count"), ({"k": None}, hip_lib.FA_EINVAL, "null k"),
    ({"v": 258}, hip_lib.FA_EINVAL, "16-byte aligned"), ({"start": None}, hip_lib.FA_EINVAL, "null start"),
    ({"k_values": 256}, hip_lib.FA_EINVAL, "go together"), ({"k_stride": _i64(1024, 512, 32, 1)}, hip_lib.FA_EINVAL, "row stride 32 of k"),
    ({"layer": 1}, hip_lib.FA_EINVAL, "layer 1 of 1"), ({"layer": -1}, hip_lib.FA_EINVAL, "layer -1"),
])
def test_append_refusals(over, code, needle):
    assert hip_lib.load().kv8_append(ctypes.byref(_append(**over)), None) == code
    assert needle in hip_lib.last_error()


@pytest.mark.parametrize("over,code,needle", [
    ({"H": 3}, hip_lib.FA_EINVAL, "multiple of kv heads"), ({"M": -1}, hip_lib.FA_EINVAL, "invalid sizes"),
    ({"sm_scale": float("nan")}, hip_lib.FA_EINVAL, "sm_scale"), ({"splits": 0}, hip_lib.FA_EINVAL, "splits"),
    ({"splits": 4097}, hip_lib.FA_EINVAL, "splits"), ({"q": None}, hip_lib.FA_EINVAL, "null q"),
    ({"o": 260}, hip_lib.FA_EINVAL, "o must be 8-byte aligned"), ({"start": None}, hip_lib.FA_EINVAL, "null start"),
    ({"splits": 2}, hip_lib.FA_EWORKSPACE, "split workspace"), ({"M": 1 << 30, "H": 8}, hip_lib.FA_EINVAL, "too many query rows"),
    ({"layer": 2}, hip_lib.FA_EINVAL, "layer 2"),
])
def test_attend_refusals(over, code, needle):
    assert hip_lib.load().kv8_attend(ctypes.byref(_attend(**over)), None) == code
    assert needle in hip_lib.last_error()


def test_page_refusals():
    lib = hip_lib.load()
    for over, code, needle in (({"rows": -1}, hip_lib.FA_EINVAL, "row count"), ({"start": None}, hip_lib.FA_EINVAL, "null start"),
                               ({"missing": None}, hip_lib.FA_EINVAL, "null missing"), ({"workspace": 264}, hip_lib.FA_EINVAL, "aligned"),
                               ({"workspace": None}, hip_lib.FA_EWORKSPACE, "reserve workspace"),
                               ({"workspace_bytes": 8}, hip_lib.FA_EWORKSPACE, "got 8")):
        assert lib.kv8_reserve(ctypes.byref(_reserve(**over)), None) == code
        assert needle in hip_lib.last_error()
    for over, code, needle in (({"used": None}, hip_lib.FA_EINVAL, "null used"),
                               ({"workspace": None}, hip_lib.FA_EWORKSPACE, "compact workspace")):
        assert lib.kv8_compact(ctypes.byref(_compact(**over)), None) == code
        assert needle in hip_lib.last_error()
    assert lib.kv8_fork(ctypes.byref(_cache()), None, None) == lib.kv8_truncate(ctypes.byref(_cache()), None, None) == hip_lib.FA_EINVAL
    assert lib.kv8_fork(ctypes.byref(_cache(B=kv8.MAX_FORK + 1)), 256, None) == hip_lib.FA_ENOTSUP
    assert "fork of 16385" in hip_lib.last_error()


def test_grids_that_hip_does_not_take():
    lib = hip_lib.load()
    rows = _i64(1 << 40, 1 << 35, 64, 1)
    wide = _cache(B=64, H_kv=1 << 20, page_stride=1 << 40)
    assert lib.kv8_append(ctypes.byref(_append(wide, rows=1 << 10, k_stride=rows, v_stride=rows)), None) == hip_lib.FA_EINVAL
    assert "cache append grid too large" in hip_lib.last_error()
    many = _attend(_cache(B=1 << 18, H_kv=1), H=16, M=1, splits=33, workspace=256, workspace_bytes=1 << 60)
    assert lib.kv8_attend(ctypes.byref(many), None) == hip_lib.FA_EINVAL
    assert "cache merge grid too large" in hip_lib.last_error()
    chunks = _attend(_cache(B=1 << 14, H_kv=1), H=1, M=1 << 12, splits=512, workspace=256, workspace_bytes=1 << 60)
    assert lib.kv8_attend(ctypes.byref(chunks), None) == hip_lib.FA_EINVAL
    assert "cache join grid too large" in hip_lib.last_error()


def test_compact_needs_the_counts_without_sequences_too():
    lib = hip_lib.load()
    for over in ({"refs": None}, {"data": None}):
        assert lib.kv8_compact(ctypes.byref(_compact(_cache(B=0, **over))), None) == hip_lib.FA_EINVAL
        assert "null cache" in hip_lib.last_error()


def test_empty_calls_do_nothing():
    lib = hip_lib.load()
    assert lib.kv8_append(None, None) == lib.kv8_attend(None, None) == hip_lib.FA_EINVAL
    assert lib.kv8_reserve(None, None) == lib.kv8_compact(None, None) == hip_lib.FA_EINVAL
    assert lib.kv8_fork(None, None, None) == lib.kv8_truncate(None, None, None) == hip_lib.FA_EINVAL
    assert lib.kv8_append(ctypes.byref(_append(rows=0)), None) == lib.kv8_attend(ctypes.byref(_attend(M=0)), None) == hip_lib.FA_OK
    for f in (lib.kv8_fork, lib.kv8_truncate):
        assert f(ctypes.byref(_cache(B=0)), None, None) == hip_lib.FA_OK
    assert lib.kv8_append(ctypes.byref(_append(_cache(B=0))), None) == hip_lib.FA_OK
    assert lib.kv8_page_bytes(2, 64, 64) == 2 * 2 * 64 * 64 + 128 and lib.kv8_page_bytes(0, 64, 64) == 0
    assert lib.kv8_page_bytes(64, 256, 128) == 2 * 64 * 256 * 128 + 2 * 64 * 8
    assert lib.kv8_attend_workspace_bytes(2, 4, 2, 3, 64, 5) == 5 * 24 * (64 * 4 + 8)
    assert lib.kv8_attend_workspace_bytes(2, 4, 2, 300, 64, 5) == 2 * 5 * 128 * (64 * 4 + 8) + 8 * 2 * 2 * 5
    assert lib.kv8_attend_workspace_bytes(1, 1, 1, 1, 64, 1) == lib.kv8_reserve_workspace_bytes(None, 1) == 0


def test_python_refusals_without_a_gpu():
    make = lambda *a, **k: kv8.Kv8Cache(*a, **{"dtype": torch.float16, **k})  # noqa: E731
    with pytest.raises(ValueError, match="lives on a GPU"):
        make(1, 1, 8, 64, device="cpu")
    for bad in ({"dtype": torch.float32}, {"page_size": 16}, {"page_size": 96}, {"pages": (1 << 30) + 1}):
        with pytest.raises(hip_lib.FaUnsupportedError):
            make(1, 1, 8, 64, **bad)
    for sizes in ((1, 1, 8, 96), (1, 1, (1 << 30) + 1, 64), (1 << 20, 1, 1 << 20, 64)):
        with pytest.raises(hip_lib.FaUnsupportedError):
            make(*sizes)
    for sizes, more in (((1, 1, 0, 64), {}), ((1, 0, 8, 64), {}), ((-1, 1, 8, 64), {}), ((1, 1, 8, 64), {"pages": 0}), ((1, 1, 8, 64), {"layers": 0})):
        with pytest.raises(ValueError, match="invalid cache sizes"):
            make(*sizes, **more)


def test_splits_rule():
    """Grids that fill the chip are not split; no split has less than 256 keys of a full cache."""
    assert kv8.choose_splits(256, 32, 8, 1, 128, 65536) == 1
    assert kv8.choose_splits(1, 32, 8, 1, 128, 255) == 1
    for B, H, Hk, M, D, cap in ((1, 32, 8, 1, 128, 8192), (1, 12, 2, 4, 128, 100000), (2, 28, 4, 509, 128, 16384), (1, 1, 1, 1, 64, 1 << 20)):
        n = kv8.choose_splits(B, H, Hk, M, D, cap)
        blocks = B * Hk * -(-M * (H // Hk) // 128) if M * (H // Hk) > 32 else 1
        assert 1 <= n <= max(1, -(-cap // 256)) * blocks and n <= 4096


def test_the_model_follows_the_format():
    """Codes as torch's e4m3 type has them; a block's largest magnitude lands in (224, 448] steps, the others on the
    nearest code."""
    assert torch.equal(kv8_model.VALUES.nan_to_num(999), torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().nan_to_num(999))
    gen = torch.Generator().manual_seed(0)
    for dtype in (torch.float16, torch.bfloat16):
        for size in (1e-6, 0.3, 7.0, 2000.0):
            x = (torch.randn(32, 64, generator=gen) * size).to(dtype).double()
            e, c = kv8_model.encode_block(x, dtype)
            step = math.ldexp(1.0, e - 127)
            if kv8_model.RANGE[dtype][0] < e:
                assert 224 < float(x.abs().max()) / step <= 448
            y = (x / step).float().to(torch.float8_e4m3fn)
            assert torch.equal(kv8_model.VALUES[c.long()], y.double())
    e, c = kv8_model.encode_block(torch.full((32, 64), math.inf, dtype=torch.float64), torch.float16)
    assert e == 112 and (c == 127).all()
    assert kv8_model.encode_block(torch.full((32, 64), 1.75, dtype=torch.float64), torch.float16)[0] == 127 - 8
    assert kv8_model.encode_block(torch.full((32, 64), 1.7501, dtype=torch.float64), torch.float16)[0] == 127 - 7
    assert callable(flash_atten.sdpa_kv8)
