// Argument checks and the launch that the C entries share.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>

#include "fa_kernels.h"
#include "../../include/fa_gfx950.h"

namespace fa {
namespace abi {

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

inline int check_type(int dtype, int D) {
  if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16)
    return fail(FA_ENOTSUP, "unsupported dtype code %d (fp16=0, bf16=1)", dtype);
  if (D != 64 && D != 128 && D != 256) return fail(FA_ENOTSUP, "head dim D=%d is not built (64, 128, 256)", D);
  return FA_OK;
}

// A [batch, heads, rows, D] operand: unit stride along D, rows that do not overlap, 16-byte alignment (`step`
// elements), and 256 rows inside a 32-bit byte offset.
inline int check_tensor(const char* name, const void* ptr, const int64_t* stride, int D, int step) {
  if (ptr == nullptr) return fail(FA_EINVAL, "null %s pointer", name);
  if (stride[3] != 1) return fail(FA_EINVAL, "head-dim stride of %s must be 1", name);
  if (!aligned(ptr, (uintptr_t)step * 2)) return fail(FA_EINVAL, "%s must be %d-byte aligned", name, step * 2);
  for (int i = 0; i < 3; ++i)
    if (stride[i] % step) return fail(FA_EINVAL, "strides of %s must be multiples of %d elements", name, step);
  if (stride[2] < D || stride[2] > (1 << 22))
    return fail(FA_EINVAL, "row stride %lld of %s is outside %d .. 2^22", (long long)stride[2], name, D);
  return FA_OK;
}

inline int check_scale(float scale) {
  if (!std::isfinite(scale * 1.4426950408889634f) || scale <= 0.f)
    return fail(FA_EINVAL, "sm_scale must be positive and finite, got %g", (double)scale);
  return FA_OK;
}

inline void copy3(int64_t* dst, const int64_t* src) { std::memcpy(dst, src, 3 * sizeof(int64_t)); }

inline int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// HIP takes less than 2^32 threads along a dimension. Every entry asks before its first launch.
inline int check_grid(int64_t blocks, int threads, const char* what) {
  if (blocks > 0xffffffffLL / threads)
    return fail(FA_EINVAL, "%s grid too large (%lld workgroups of %d)", what, (long long)blocks, threads);
  return FA_OK;
}

inline int launch(const void* fn, int64_t blocks, int64_t y, int threads, void* params, void* stream, const char* what) {
  void* args[] = {params};
  const hipError_t err = hipLaunchKernel(fn, dim3((unsigned)blocks, (unsigned)y), dim3((unsigned)threads), args, 0,
                                         static_cast<hipStream_t>(stream));
  if (err != hipSuccess) return fail(FA_EHIP, "%s launch failed: %s", what, hipGetErrorString(err));
  return FA_OK;
}

}  // namespace abi
}  // namespace fa
