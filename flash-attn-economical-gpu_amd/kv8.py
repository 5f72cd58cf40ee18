"""Paged key/value cache held in 8 bits, for serving: sequences that come and go, drafts, beams that share a prompt.

A cached channel takes one byte (e4m3: 4 exponent bits, 3 mantissa bits), and 32 tokens of a kv head share a
power-of-two scale byte, a format that gfx950 converts to fp16 and bf16 in hardware. Tokens live in pages of
`page_size` that sequences take from a common pool; one page table serves all layers. The caller keeps the lengths, as
int32 tensors on the GPU, and every call takes them from there, so a decode loop needs no host round trip and can be
captured into a HIP graph:

    cache = Kv8Cache(B, H_kv, capacity, D, dtype=torch.bfloat16, pages=4096, layers=L)
    cache.reserve(start, k.shape[2], count=count)                       # pages for the new tokens, copied where shared
    cache.append(k, v, start, count=count, layer=i)                     # tokens start[b] .. start[b] + count[b]
    out = flash_atten.sdpa_kv8(q, cache, start, count=count, layer=i)   # the same tokens' queries
    start += count
    cache.fork(parent)                                                  # sequence b goes on from sequence parent[b]
    cache.truncate(length)                                              # what lies behind length[b] tokens is given up

Calls that change a cache (its pages, its table) are ordered by the caller, as writes of any tensor are; the state is
the table and the page counts, and a call's result depends on nothing else, so repeated runs give the same bits.

The reference has no cache (its models keep one in full precision); nothing here has a counterpart in it.
"""
from __future__ import annotations

import ctypes
import functools

import torch

import hip_lib
from kv4 import _form, _plans, keep_plan

BLOCK = 32  # tokens that share a scale
PAGE_SIZES = (32, 64, 128, 256)
MAX_CAPACITY = 1 << 30  # KV8_MAX_CAPACITY in include/fa_gfx950.h
MAX_FORK = 16384  # KV8_MAX_FORK


@functools.lru_cache(maxsize=4096)
def choose_splits(B: int, H: int, H_kv: int, M: int, D: int, capacity: int) -> int:
    """Parts that a sequence's keys are cut into on average (up to 32 query rows to a kv head), or workgroups that share
    all the work (more rows): as many workgroups as the chip holds, none with less than 256 keys of a full cache."""
    return int(hip_lib.load().kv8_attend_splits(B, H, H_kv, M, D, capacity))


class Kv8Cache:
    """8-bit keys and values of `batch` sequences of up to `capacity` tokens, in `pages` pages of `page_size` tokens
    (without a number: as many as all sequences can need without sharing any)."""

    def __init__(self, batch: int, kv_heads: int, capacity: int, head_dim: int, *, dtype: torch.dtype,
                 pages: int | None = None, page_size: int = 64, layers: int = 1,
                 device: torch.device | str = "cuda") -> None:
        hip_lib.dtype_code(dtype)
        if head_dim not in (64, 128, 256):
            raise hip_lib.FaUnsupportedError(f"head dim {head_dim} is not built (64, 128, 256)")
        if page_size not in PAGE_SIZES:
            raise hip_lib.FaUnsupportedError(f"pages of {page_size} tokens are not built {PAGE_SIZES}")
        if batch < 0 or kv_heads < 1 or capacity < 1 or layers < 1 or (pages is not None and pages < 1):
            raise ValueError(f"invalid cache sizes batch={batch} kv_heads={kv_heads} capacity={capacity} layers={layers} "
                             f"pages={pages}")
        if capacity > MAX_CAPACITY:
            raise hip_lib.FaUnsupportedError(f"capacity {capacity} is beyond {MAX_CAPACITY}")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"an 8-bit cache lives on a GPU, got device {device}")
        columns = -(-capacity // page_size)
        if batch * columns > 1 << 30:
            raise hip_lib.FaUnsupportedError(f"a page table of {batch} x {columns} entries is beyond 2^30")
        pages = max(1, batch * columns) if pages is None else pages
        if pages > MAX_CAPACITY:
            raise hip_lib.FaUnsupportedError(f"{pages} pages are beyond {MAX_CAPACITY}")
        stride = hip_lib.kv8_page_bytes(kv_heads, page_size, head_dim)
        data = torch.zeros(layers, pages, stride, dtype=torch.uint8, device=device)
        self._data = data
        self._table = torch.full((batch, columns), -1, dtype=torch.int32, device=device)
        self._refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.batch, self.kv_heads, self.capacity, self.head_dim = batch, kv_heads, capacity, head_dim
        self.pages, self.page_size, self.layers, self.dtype, self.device = pages, page_size, layers, dtype, data.device
        half, blocks = page_size * head_dim, page_size // BLOCK
        lead = (layers, pages, kv_heads)
        strides = data.stride()[:2]
        self._codes = tuple(data.as_strided((*lead, page_size, head_dim), (*strides, 2 * half, head_dim, 1), i * half)
                            for i in range(2))
        self._scales = tuple(data.as_strided((*lead, blocks), (*strides, 2 * blocks, 2), 2 * kv_heads * half + i)
                             for i in range(2))
        c = self._args = hip_lib.Kv8CacheArgs()
        c.data, c.table, c.refs = data.data_ptr(), self._table.data_ptr(), self._refs.data_ptr()
        c.layer_stride, c.page_stride = strides
        c.B, c.H_kv, c.D, c.dtype = batch, kv_heads, head_dim, hip_lib.dtype_code(dtype)
        c.page, c.pages, c.columns, c.capacity, c.layers = page_size, pages, columns, capacity, layers
        self._form = ("kv8", batch, kv_heads, capacity, head_dim, pages, page_size, layers, dtype, self.device)

    # The state. It may be written in place, not replaced: `table` [batch, columns] holds the page of each page_size
    # tokens of a sequence, or -1; `refs` [pages] the number of entries that name a page (0: free). Codes are
    # [layers, pages, kv heads, page_size, D] e4m3 bytes, scale bytes e [layers, pages, kv heads, page_size / 32]
    # stand for 2^(e - 127).
    @property
    def table(self) -> torch.Tensor:
        return self._table

    @property
    def refs(self) -> torch.Tensor:
        return self._refs

    @property
    def k_codes(self) -> torch.Tensor:
        return self._codes[0]

    @property
    def v_codes(self) -> torch.Tensor:
        return self._codes[1]

    @property
    def k_scales(self) -> torch.Tensor:
        return self._scales[0]

    @property
    def v_scales(self) -> torch.Tensor:
        return self._scales[1]

    def nbytes(self) -> int:
        return self._data.numel()

    def reserve(self, start: torch.Tensor, rows: int, *, count: torch.Tensor | None = None) -> torch.Tensor:
        """Pages that `append` may write for tokens start[b] .. start[b] + n - 1, n = min(rows, count[b]) (rows
        without a count). In order of sequence and token, an entry without a page takes the lowest free page; one whose
        page has other holders takes the lowest free page and a copy of it in all layers (but for the last such entry
        of a page whose holders are all among them, which keeps it). Returns how many pages were wanting, int32 [1] on
        the GPU: those entries stay as they are, and appends to them are dropped. So are appends to a page that its last
        holder keeps while one of the others still waits: the page has two holders until a later `reserve` finds
        it a free one."""
        if not isinstance(rows, int) or rows < 0:
            raise ValueError(f"rows must be a number of tokens, got {rows!r}")
        rows = min(rows, 2 ** 31 - 1)
        start, count = self.positions(start, count)
        missing = torch.empty(1, dtype=torch.int32, device=self.device)
        workspace = torch.empty(hip_lib.kv8_reserve_workspace_bytes(self._form, self._args, rows), dtype=torch.uint8,
                                device=self.device)
        hip_lib.kv8_reserve(self._args, start, count, rows, missing, workspace, self.device)
        return missing

    def append(self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, *, count: torch.Tensor | None = None,
               layer: int = 0, return_values: bool = False) -> tuple[torch.Tensor, torch.Tensor] | None:
        """Rows t < count[b] (all without a count) of k and v [batch, kv heads, rows, D] become tokens start[b] + t of
        a layer. The 32-token blocks that get tokens are encoded anew, from what their tokens before start[b] stand for
        and the new rows; their tokens behind the new ones become zeros, so start[b] + count[b] is the sequence's
        length from here on. Rows outside the capacity, or whose page is missing or shared, are dropped (`reserve`
        comes first). With return_values, returns what the rows now stand for (zeros in rows that were not written), in
        k's type, for a layer that goes on with the values its later steps will see. They take no part in autograd."""
        self._layer(layer)  # before the look-up: 1.0 is equal to 1, and no layer
        key = (self._form, _form(k), _form(v), _form(start), None if count is None else _form(count), layer,
               bool(return_values))
        plan = _plans.get(key)
        if plan is None or (k.data_ptr() | v.data_ptr()) & 15:
            k, v, start, count = self._append_operands(k, v, start, count)
            values = (hip_lib.dense_like(k), hip_lib.dense_like(v)) if return_values else (None, None)
            plan = hip_lib.kv8_append_plan(k, v, *values, layer=layer)
            if key == (self._form, _form(k), _form(v), _form(start), None if count is None else _form(count), layer,
                       bool(return_values)):  # nothing had to be copied: calls of this form take the short way
                keep_plan(key, plan)
        else:
            values = (hip_lib.dense_like(k), hip_lib.dense_like(v)) if return_values else (None, None)
        hip_lib.kv8_append_planned(plan, self._args, k, v, start, count, *values)
        return values if return_values else None

    def fork(self, parent: torch.Tensor) -> None:
        """Sequence b goes on from what sequence parent[b] (int32 [batch] on the GPU) held before the call: it names the
        same pages, and gives up its own. parent[b] = b changes nothing, a parent outside the batch (-1) leaves the
        sequence empty. No page is copied: `reserve` does that where a shared one is about to be written."""
        hip_lib.kv8_fork(self._args, self._lengths("parent", parent), self.device)

    def truncate(self, length: torch.Tensor) -> None:
        """Pages that hold none of sequence b's first length[b] (int32 [batch] on the GPU) tokens are given up; 0 frees
        the sequence."""
        hip_lib.kv8_truncate(self._args, self._lengths("length", length), self.device)

    def compact(self) -> torch.Tensor:
        """Pages in use move to the front of the pool, in all layers, and the table follows. Returns their number, int32
        [1] on the GPU."""
        used = torch.empty(1, dtype=torch.int32, device=self.device)
        workspace = torch.empty(hip_lib.kv8_compact_workspace_bytes(self._args), dtype=torch.uint8,
                                device=self.device)
        hip_lib.kv8_compact(self._args, used, workspace, self.device)
        return used

    def _append_operands(self, k, v, start, count):
        """append's arguments, checked, and copied where the kernels cannot read them as they lie."""
        for name, t in (("k", k), ("v", v)):
            if not isinstance(t, torch.Tensor):
                raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
        shape = (self.batch, self.kv_heads, k.shape[2] if k.dim() == 4 else -1, self.head_dim)
        for name, t in (("k", k), ("v", v)):
            if tuple(t.shape) != shape or t.dtype != self.dtype or t.device != self.device:
                raise ValueError(f"{name} must be {self.dtype} [{self.batch}, {self.kv_heads}, rows, {self.head_dim}] on "
                                 f"{self.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
        start, count = self.positions(start, count)
        return hip_lib.operand(k, "k"), hip_lib.operand(v, "v"), start, count

    def _layer(self, layer: int) -> None:
        if not isinstance(layer, int) or not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer!r} of a cache with {self.layers}")

    def _lengths(self, name: str, t: torch.Tensor) -> torch.Tensor:
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (self.batch,) or t.device != self.device:
            got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
            raise ValueError(f"{name} must be an int32 tensor [{self.batch}] on {self.device}, got {got}")
        return t.contiguous()

    def positions(self, start: torch.Tensor, count: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor | None]:
        """start and count as the kernels read them; ValueError if they are anything but int32 [batch] here."""
        return self._lengths("start", start), None if count is None else self._lengths("count", count)


__all__ = ["BLOCK", "MAX_CAPACITY", "MAX_FORK", "PAGE_SIZES", "Kv8Cache", "choose_splits"]
