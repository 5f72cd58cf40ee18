"""Calls whose grids HIP does not take (2^32 threads along a dimension) are refused by the C entries before the first
launch, so that no error of the runtime is left behind and no output is half written (no GPU needed)."""
from __future__ import annotations

import ctypes

import hip_lib
from test_operators_cpu import _append, _attend, _bwd, _cache, _i64


def _refused(code, what):
    assert code == hip_lib.FA_EINVAL
    assert f"{what} grid too large" in hip_lib.last_error()


def test_append():
    """2^29 rows of 64 channels are 2^32 threads of 8 channels."""
    cache = _cache(H_kv=1, capacity=1 << 30, rows=1 << 30, D=64)
    rows = _i64(1 << 40, 1 << 35, 64, 1)
    a = _append(cache, rows=1 << 29, k_stride=rows, v_stride=rows)
    _refused(hip_lib.load().kv4_append(ctypes.byref(a), None), "cache append")


def test_merge():
    """Sixteen waves to a row: 2^22 rows are 2^32 threads; the attention kernel before it is not launched either."""
    cache = _cache(B=64, H_kv=1, code_stride=_i64(4096, 2048), scale_stride=_i64(256, 128))
    a = _attend(cache, H=1, M=1 << 16, splits=33, workspace=256, workspace_bytes=1 << 60, q_stride=_i64(1 << 22, 1 << 22, 64, 1),
                o_stride=_i64(1 << 22, 1 << 22, 64, 1))
    _refused(hip_lib.load().kv4_attend(ctypes.byref(a), None), "cache merge")


def test_backward():
    """2^30 query rows: 2^24 blocks of 64 rows for their terms."""
    a = _bwd(B=1 << 10, H=1 << 10, H_kv=1 << 10, M=1 << 10, N=64, workspace_bytes=1 << 60)
    _refused(hip_lib.load().fa_bwd(ctypes.byref(a), None), "row-term")
