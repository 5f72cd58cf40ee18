"""Refusals of the paged 8-bit cache's C entries that come before any launch (no GPU needed)."""
from __future__ import annotations

import ctypes

import pytest

import hip_lib
from test_kv8_cpu import _append, _attend, _cache, _compact, _reserve

PAGE = 16512  # bytes of _cache()'s pages, of which it has 8


def _calls(c):
    lib = hip_lib.load()
    yield lambda: lib.kv8_append(ctypes.byref(_append(c, rows=-1)), None), "row count"
    yield lambda: lib.kv8_attend(ctypes.byref(_attend(c, M=-1)), None), "invalid sizes"
    yield lambda: lib.kv8_reserve(ctypes.byref(_reserve(c, rows=-1)), None), "row count"
    yield lambda: lib.kv8_compact(ctypes.byref(_compact(c, used=None)), None), "null used"
    yield lambda: lib.kv8_fork(ctypes.byref(c), None, None), "null parent"
    yield lambda: lib.kv8_truncate(ctypes.byref(c), None, None), "null length"


@pytest.mark.parametrize("layers,pages,page_stride,layer_stride,fits", [
    (2, 8, PAGE, 8 * PAGE, True), (2, 8, PAGE, 8 * PAGE - 16, False), (2, 8, PAGE, 0, False), (2, 8, PAGE, PAGE, False),
    (3, 8, 3 * PAGE, PAGE, True), (3, 8, 3 * PAGE - 16, PAGE, False), (3, 8, 3 * PAGE, PAGE - 16, False),  # a page's layers together
    (2, 8, PAGE, -8 * PAGE, False), (2, 8, 1 << 60, 1 << 60, False), (2, 8, 1 << 62, 1 << 62, False), (2, 8, 1 << 62, PAGE, True),
    (2, 1, 0, PAGE, True), (2, 1, 0, PAGE - 16, False), (1, 8, PAGE, 0, True), (1 << 30, 8, PAGE, 8 * PAGE, True),
])
def test_layers_that_overlap_are_refused(layers, pages, page_stride, layer_stride, fits):
    c = _cache(layers=layers, pages=pages, page_stride=page_stride, layer_stride=layer_stride)
    for call, later in _calls(c):
        assert call() == hip_lib.FA_EINVAL
        assert (later if fits else "overlap") in hip_lib.last_error()
