"""Key/value cache held in 4 bits, for decode and for prompts that arrive in chunks.

A cached row of D channels takes 17/32 byte per channel: 4-bit codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign)
and one power-of-two scale for 32 channels, a format that gfx950 converts to fp16 and bf16 in hardware. The
cache is [batch, kv heads, capacity, D]; the caller keeps the lengths, as int32 tensors on the GPU, so a decode
loop needs no host round trip and can be captured into a HIP graph:

    cache = Kv4Cache(B, H_kv, capacity, D, dtype=torch.bfloat16)
    cache.append(k, v, start, count=count)                              # rows start[b] .. start[b] + count[b]
    out = flash_atten.sdpa_kv4(q, cache, start, count=count)            # the same rows' queries
    start += count

The reference has no cache (its models keep one in full precision); nothing here has a counterpart in it.
"""
from __future__ import annotations

import ctypes
import functools

import torch

import hip_lib

BLOCK = 32  # channels that share a scale
MAX_CAPACITY = 1 << 30  # KV4_MAX_CAPACITY in include/fa_gfx950.h


# Argument blocks by the values they depend on (shapes, strides, types, devices, flags): the checks and filling a
# block field by field are most of a call's host time, which single-token calls would wait for. No tensor or
# address is kept.
_plans: dict[tuple, object] = {}
_MAX_PLANS = 4096


def keep_plan(key: tuple, plan) -> None:
    if len(_plans) >= _MAX_PLANS:
        _plans.clear()
    _plans[key] = plan


def _form(t) -> tuple:
    return (t.shape, t.stride(), t.dtype, t.device) if isinstance(t, torch.Tensor) else (type(t),)


@functools.lru_cache(maxsize=4096)
def choose_splits(B: int, H: int, H_kv: int, M: int, D: int, capacity: int) -> int:
    """Parts that a sequence's keys are cut into on average: as many workgroups as the chip holds, none with less
    than 256 keys of a full cache."""
    return int(hip_lib.load().kv4_attend_splits(B, H, H_kv, M, D, capacity))


class Kv4Cache:
    """4-bit keys and values of `batch` sequences of up to `capacity` tokens."""

    def __init__(self, batch: int, kv_heads: int, capacity: int, head_dim: int, *, dtype: torch.dtype,
                 device: torch.device | str = "cuda") -> None:
        hip_lib.dtype_code(dtype)
        if head_dim not in (64, 128, 256):
            raise hip_lib.FaUnsupportedError(f"head dim {head_dim} is not built (64, 128, 256)")
        if batch < 0 or kv_heads < 1 or capacity < 1:
            raise ValueError(f"invalid cache sizes batch={batch} kv_heads={kv_heads} capacity={capacity}")
        if capacity > MAX_CAPACITY:
            raise hip_lib.FaUnsupportedError(f"capacity {capacity} is beyond {MAX_CAPACITY}")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"a 4-bit cache lives on a GPU, got device {device}")
        rows = -(-capacity // 32) * 32  # the kernels read whole 32-row tiles
        full = [torch.zeros(batch, kv_heads, rows, n, dtype=torch.uint8, device=device)
                for n in (head_dim // 2, head_dim // BLOCK) * 2]
        self._buffers = tuple(t[:, :, :capacity] for t in full)
        self.batch, self.kv_heads, self.capacity, self.head_dim = batch, kv_heads, capacity, head_dim
        self.dtype, self.device = dtype, full[0].device
        c = self._args = hip_lib.Kv4CacheArgs()
        c.k_codes, c.k_scales, c.v_codes, c.v_scales = (t.data_ptr() for t in full)
        c.code_stride = (ctypes.c_int64 * 2)(*full[0].stride()[:2])
        c.scale_stride = (ctypes.c_int64 * 2)(*full[1].stride()[:2])
        c.B, c.H_kv, c.D, c.dtype = batch, kv_heads, head_dim, hip_lib.dtype_code(dtype)
        c.rows, c.capacity = rows, capacity
        self._form = (batch, kv_heads, capacity, head_dim, dtype, self.device)

    # The buffers, [batch, kv heads, capacity, bytes] (two codes to a byte, channel 2i in the low half of byte
    # i; scale byte e stands for 2^(e - 127), 255 for NaN). They may be written in place, not replaced.
    @property
    def k_codes(self) -> torch.Tensor:
        return self._buffers[0]

    @property
    def k_scales(self) -> torch.Tensor:
        return self._buffers[1]

    @property
    def v_codes(self) -> torch.Tensor:
        return self._buffers[2]

    @property
    def v_scales(self) -> torch.Tensor:
        return self._buffers[3]

    def nbytes(self) -> int:
        return sum(t.numel() for t in self._buffers)

    def append(self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, *, count: torch.Tensor | None = None,
               return_values: bool = False) -> tuple[torch.Tensor, torch.Tensor] | None:
        """Rows t < count[b] (all without a count) of k and v [batch, kv heads, rows, D] become tokens
        start[b] + t. Rows outside the capacity are dropped; what is not written stays as it is. With
        return_values, returns what the rows now stand for (zeros in rows that were not written), in k's type,
        for a layer that goes on with the values its later steps will see."""
        key = (self._form, _form(k), _form(v), _form(start), None if count is None else _form(count), bool(return_values))
        plan = _plans.get(key)
        if plan is None or (k.data_ptr() | v.data_ptr()) & 15:
            k, v, start, count = self._append_operands(k, v, start, count)
            values = (hip_lib.dense_like(k), hip_lib.dense_like(v)) if return_values else (None, None)
            plan = hip_lib.kv4_append_plan(k, v, *values)
            if key == (self._form, _form(k), _form(v), _form(start), None if count is None else _form(count),
                       bool(return_values)):  # nothing had to be copied: calls of this form take the short way
                keep_plan(key, plan)
        else:
            values = (hip_lib.dense_like(k), hip_lib.dense_like(v)) if return_values else (None, None)
        hip_lib.kv4_append_planned(plan, self._args, k, v, start, count, *values)
        return values if return_values else None

    def _append_operands(self, k, v, start, count):
        """append's arguments, checked, and copied where the kernels cannot read them as they lie."""
        shape = (self.batch, self.kv_heads, k.shape[2] if k.dim() == 4 else -1, self.head_dim)
        for name, t in (("k", k), ("v", v)):
            if tuple(t.shape) != shape or t.dtype != self.dtype or t.device != self.device:
                raise ValueError(f"{name} must be {self.dtype} [{self.batch}, {self.kv_heads}, rows, {self.head_dim}] on "
                                 f"{self.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
        start, count = self.positions(start, count)
        return hip_lib.operand(k, "k"), hip_lib.operand(v, "v"), start, count

    def positions(self, start: torch.Tensor, count: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor | None]:
        """start and count as the kernels read them; ValueError if they are anything but int32 [batch] here."""
        out = []
        for name, t in (("start", start), ("count", count)):
            if t is None and name == "count":
                out.append(None)
                continue
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (self.batch,) or t.device != self.device:
                got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
                raise ValueError(f"{name} must be an int32 tensor [{self.batch}] on {self.device}, got {got}")
            out.append(t.contiguous())
        return out[0], out[1]


__all__ = ["BLOCK", "MAX_CAPACITY", "Kv4Cache", "choose_splits"]
