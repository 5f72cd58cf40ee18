// C ABI of attention's backward pass and of the 4-bit key/value cache (declared in include/fa_gfx950.h):
// argument validation and launches on the caller's stream.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>

#include "fa_kernels.h"
#include "../../include/fa_gfx950.h"

namespace {

using fa::fail;
using fa::ok;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

const fa::BwdKernelEntry* find_bwd(int dtype, int D) {
  int n = 0;
  const fa::BwdKernelEntry* e = fa::fa_bwd_registry(&n);
  for (int i = 0; i < n; ++i)
    if (e[i].dtype == dtype && e[i].D == D) return &e[i];
  return nullptr;
}

const fa::Kv4KernelEntry* find_kv4(int dtype, int D) {
  int n = 0;
  const fa::Kv4KernelEntry* e = fa::kv4_registry(&n);
  for (int i = 0; i < n; ++i)
    if (e[i].dtype == dtype && e[i].D == D) return &e[i];
  return nullptr;
}

int check_type(int dtype, int D) {
  if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16)
    return fail(FA_ENOTSUP, "unsupported dtype code %d (fp16=0, bf16=1)", dtype);
  if (D != 64 && D != 128 && D != 256) return fail(FA_ENOTSUP, "head dim D=%d is not built (64, 128, 256)", D);
  return FA_OK;
}

// A [batch, heads, rows, D] operand: unit stride along D, rows that do not overlap, 16-byte alignment (`step`
// elements), and 256 rows inside a 32-bit byte offset.
int check_tensor(const char* name, const void* ptr, const int64_t* stride, int D, int step) {
  if (ptr == nullptr) return fail(FA_EINVAL, "null %s pointer", name);
  if (stride[3] != 1) return fail(FA_EINVAL, "head-dim stride of %s must be 1", name);
  if (!aligned(ptr, (uintptr_t)step * 2)) return fail(FA_EINVAL, "%s must be %d-byte aligned", name, step * 2);
  for (int i = 0; i < 3; ++i)
    if (stride[i] % step) return fail(FA_EINVAL, "strides of %s must be multiples of %d elements", name, step);
  if (stride[2] < D || stride[2] > (1 << 22))
    return fail(FA_EINVAL, "row stride %lld of %s is outside %d .. 2^22", (long long)stride[2], name, D);
  return FA_OK;
}

int check_scale(float scale) {
  if (!std::isfinite(scale * 1.4426950408889634f) || scale <= 0.f)
    return fail(FA_EINVAL, "sm_scale must be positive and finite, got %g", (double)scale);
  return FA_OK;
}

void copy3(int64_t* dst, const int64_t* src) { std::memcpy(dst, src, 3 * sizeof(int64_t)); }

int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// HIP takes less than 2^32 threads along a dimension. Every entry asks before its first launch.
int check_grid(int64_t blocks, int threads, const char* what) {
  if (blocks > 0xffffffffLL / threads)
    return fail(FA_EINVAL, "%s grid too large (%lld workgroups of %d)", what, (long long)blocks, threads);
  return FA_OK;
}

int launch(const void* fn, int64_t blocks, int64_t y, int threads, void* params, void* stream, const char* what) {
  void* args[] = {params};
  const hipError_t err = hipLaunchKernel(fn, dim3((unsigned)blocks, (unsigned)y), dim3((unsigned)threads), args, 0,
                                         static_cast<hipStream_t>(stream));
  if (err != hipSuccess) return fail(FA_EHIP, "%s launch failed: %s", what, hipGetErrorString(err));
  return FA_OK;
}

constexpr int kBwdPrepRows = 64;

struct BwdSizes {
  int64_t row_groups, prep_blocks, vblocks, nblocks, mblocks;
  int64_t kv_splits, q_splits;
  int64_t bound_at, dk_at, dv_at, dq_at, bytes;  // workspace offsets and size
};

// How many workgroups share a block's steps. A step is a 32-row tile against a block: four products for dK/dV,
// three for dQ. The chip (256 CUs) holds `slots` workgroups; a block that is longer than an even share of all
// work (and than kMinWork, below which the sums' extra pass costs more than it gives) is split to that. One number of
// parts for all blocks of a kind, from the longest: under a causal mask the shorter blocks' parts are shorter.
BwdSizes bwd_sizes(const fa::BwdKernelEntry* e, int64_t B, int64_t H, int64_t Hkv, int64_t M, int64_t N, int64_t D,
                   bool causal) {
  constexpr int64_t kMinWork = 32;
  const int64_t slots = 256 * e->per_cu;
  BwdSizes s;
  s.prep_blocks = (M + kBwdPrepRows - 1) / kBwdPrepRows;
  s.row_groups = s.prep_blocks * (kBwdPrepRows / 32);
  s.vblocks = (N + kBwdPrepRows - 1) / kBwdPrepRows;
  s.nblocks = (N + e->block - 1) / e->block;
  s.mblocks = (M + e->block - 1) / e->block;
  const int64_t qt = (M + 31) / 32, kt = (N + 31) / 32;
  const int64_t kv_work = 4 * (H / Hkv) * qt, q_work = 3 * kt;  // of the longest block
  const int64_t all = B * Hkv * s.nblocks * kv_work + B * H * s.mblocks * q_work;
  int64_t even = (causal ? all / 2 : all) / slots;
  if (even < kMinWork) even = kMinWork;
  s.kv_splits = 2 * kv_work > 3 * even ? (kv_work + even - 1) / even : 1;
  s.q_splits = 2 * q_work > 3 * even ? (q_work + even - 1) / even : 1;
  int64_t at = align256(B * H * s.row_groups * 64 * 4);
  s.bound_at = at;
  at += align256((2 * B * H * s.prep_blocks + B * Hkv * s.vblocks) * 4);
  const int64_t kv_bytes = s.kv_splits > 1 ? align256(s.kv_splits * B * Hkv * N * D * 4) : 0;
  s.dk_at = at;
  s.dv_at = at + kv_bytes;
  s.dq_at = at + 2 * kv_bytes;
  s.bytes = s.dq_at + (s.q_splits > 1 ? s.q_splits * B * H * M * D * 4 : 0);
  return s;
}

int check_cache(const kv4_cache* c) {
  const int code = check_type(c->dtype, c->D);
  if (code != FA_OK) return code;
  if (c->B < 0 || c->H_kv <= 0 || c->capacity < 0)
    return fail(FA_EINVAL, "invalid cache sizes B=%d H_kv=%d capacity=%d", c->B, c->H_kv, c->capacity);
  if (c->capacity > KV4_MAX_CAPACITY)
    return fail(FA_ENOTSUP, "cache capacity %d is beyond %d", c->capacity, KV4_MAX_CAPACITY);
  if (c->rows % 32 || c->rows < c->capacity)
    return fail(FA_EINVAL, "cache rows=%d must be a multiple of 32 and at least the capacity %d", c->rows, c->capacity);
  if (c->B == 0 || c->capacity == 0) return FA_OK;
  if (!c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales) return fail(FA_EINVAL, "null cache pointer");
  if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16) || !aligned(c->k_scales, 16) || !aligned(c->v_scales, 16))
    return fail(FA_EINVAL, "cache buffers must be 16-byte aligned");
  for (int i = 0; i < 2; ++i)
    if (c->code_stride[i] % 16 || c->scale_stride[i] % 16)
      return fail(FA_EINVAL, "batch and head strides of cache buffers must be multiples of 16 bytes");
  return FA_OK;
}

// Which attention kernel takes a kv head's query rows: up to 32 the waves of a workgroup share them (and the
// cache is read once); more go chunk_rows to a workgroup.
struct Kv4Kind {
  int kind;
  int64_t row_blocks;
};
Kv4Kind kv4_kind(const fa::Kv4KernelEntry* e, int64_t rows) {
  Kv4Kind k;
  k.kind = rows <= 16 ? 0 : (rows <= 32 ? 1 : 2);
  const int64_t block = k.kind == 2 ? e->chunk_rows : 16 << k.kind;
  k.row_blocks = (rows + block - 1) / block;
  return k;
}

}  // namespace

extern "C" {

int64_t fa_bwd_workspace_bytes(int32_t B, int32_t H, int32_t H_kv, int32_t M, int32_t N, int32_t D, int32_t causal) {
  const fa::BwdKernelEntry* e = find_bwd(FA_DTYPE_F16, D);  // blocks are alike for both types
  if (e == nullptr || B <= 0 || H <= 0 || H_kv <= 0 || M < 0 || N < 0) return 0;
  return bwd_sizes(e, B, H, H_kv, M, N, D, causal != 0).bytes;
}

int fa_bwd(const fa_bwd_args* a, void* stream) {
  if (a == nullptr) return fail(FA_EINVAL, "null argument block");
  int code = check_type(a->dtype, a->D);
  if (code != FA_OK) return code;
  if (a->B < 0 || a->H <= 0 || a->H_kv <= 0 || a->M < 0 || a->N < 0)
    return fail(FA_EINVAL, "invalid sizes B=%d H=%d H_kv=%d M=%d N=%d", a->B, a->H, a->H_kv, a->M, a->N);
  if (a->H % a->H_kv != 0)
    return fail(FA_EINVAL, "query heads H=%d must be a multiple of kv heads H_kv=%d", a->H, a->H_kv);
  if ((code = check_scale(a->sm_scale)) != FA_OK) return code;
  if (a->B == 0 || (a->M == 0 && a->N == 0)) return ok();
  // without rows the gradients of K and V are zeros, without keys those of Q: the kernels write them
  if (a->M > 0) {
    if ((code = check_tensor("q", a->q, a->q_stride, a->D, 8)) != FA_OK) return code;
    if ((code = check_tensor("o", a->o, a->o_stride, a->D, 8)) != FA_OK) return code;
    if ((code = check_tensor("dout", a->dout, a->dout_stride, a->D, 8)) != FA_OK) return code;
    if ((code = check_tensor("dq", a->dq, a->dq_stride, a->D, 4)) != FA_OK) return code;
    if (a->lse == nullptr) return fail(FA_EINVAL, "null lse pointer");
  }
  if (a->N > 0) {
    if ((code = check_tensor("k", a->k, a->k_stride, a->D, 8)) != FA_OK) return code;
    if ((code = check_tensor("v", a->v, a->v_stride, a->D, 8)) != FA_OK) return code;
    if ((code = check_tensor("dk", a->dk, a->dk_stride, a->D, 4)) != FA_OK) return code;
    if ((code = check_tensor("dv", a->dv, a->dv_stride, a->D, 4)) != FA_OK) return code;
  }
  const int64_t need = fa_bwd_workspace_bytes(a->B, a->H, a->H_kv, a->M, a->N, a->D, a->causal);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need))
    return fail(FA_EWORKSPACE, "backward workspace of %lld bytes needed, got %lld", (long long)need,
                (long long)a->workspace_bytes);
  if (!aligned(a->workspace, 256)) return fail(FA_EINVAL, "workspace must be 256-byte aligned");
  const fa::BwdKernelEntry* e = find_bwd(a->dtype, a->D);
  if (e == nullptr) return fail(FA_ENOTSUP, "backward kernels for dtype=%d D=%d are not built", a->dtype, a->D);
  if (e->prep_rows != kBwdPrepRows) return fail(FA_ENOTSUP, "row-term blocks of %d rows", e->prep_rows);
  const BwdSizes s = bwd_sizes(e, a->B, a->H, a->H_kv, a->M, a->N, a->D, a->causal != 0);

  fa::BwdParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = static_cast<const uint16_t*>(a->q);
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.o = static_cast<const uint16_t*>(a->o);
  p.dout = static_cast<const uint16_t*>(a->dout);
  p.lse = a->lse;
  p.dlse = a->dlse;
  p.dq = static_cast<uint16_t*>(a->dq);
  p.dk = static_cast<uint16_t*>(a->dk);
  p.dv = static_cast<uint16_t*>(a->dv);
  copy3(p.sq, a->q_stride);
  copy3(p.sk, a->k_stride);
  copy3(p.sv, a->v_stride);
  copy3(p.so, a->o_stride);
  copy3(p.sdo, a->dout_stride);
  copy3(p.sl, a->lse_stride);
  copy3(p.sdl, a->dlse_stride);
  copy3(p.sdq, a->dq_stride);
  copy3(p.sdk, a->dk_stride);
  copy3(p.sdv, a->dv_stride);
  p.nd = static_cast<float*>(a->workspace);
  char* ws = static_cast<char*>(a->workspace);
  p.bound = reinterpret_cast<float*>(ws + s.bound_at);
  p.ws_dk = reinterpret_cast<float*>(ws + s.dk_at);
  p.ws_dv = reinterpret_cast<float*>(ws + s.dv_at);
  p.ws_dq = reinterpret_cast<float*>(ws + s.dq_at);
  p.B = a->B; p.H = a->H; p.Hkv = a->H_kv; p.M = a->M; p.N = a->N;
  p.group = a->H / a->H_kv;
  p.row_groups = (int32_t)s.row_groups;
  p.prep_blocks = (int32_t)s.prep_blocks;
  p.vblocks = a->dtype == FA_DTYPE_F16 ? (int32_t)s.vblocks : 0;
  p.nblocks = (int32_t)s.nblocks;
  p.mblocks = (int32_t)s.mblocks;
  p.kv_splits = (int32_t)s.kv_splits;
  p.q_splits = (int32_t)s.q_splits;
  p.causal = a->causal ? 1 : 0;
  p.scale = a->sm_scale;
  p.c = a->sm_scale * 1.4426950408889634f;
  const int64_t kv_total = (int64_t)a->B * a->H_kv * s.nblocks * s.kv_splits;
  const int64_t q_total = (int64_t)a->B * a->H * s.mblocks * s.q_splits;
  if (kv_total + q_total > 0x7fffffffLL || (int64_t)p.group * p.prep_blocks > 0x7fffffffLL)
    return fail(FA_EINVAL, "backward grid too large (%lld workgroups)", (long long)(kv_total + q_total));
  p.kv_total = (int32_t)kv_total;
  p.q_total = (int32_t)q_total;
  const int64_t prep = (int64_t)a->B * a->H * p.prep_blocks + (int64_t)a->B * a->H_kv * p.vblocks;
  const int64_t sums = ((s.kv_splits > 1 ? 2 * (int64_t)a->B * a->H_kv * a->N : 0) +
                        (s.q_splits > 1 ? (int64_t)a->B * a->H * a->M : 0)) * (a->D / 4);
  if ((code = check_grid(prep, 256, "row-term")) != FA_OK || (code = check_grid(kv_total + q_total, 256, "backward")) != FA_OK ||
      (code = check_grid((sums + 255) / 256, 256, "gradient sum")) != FA_OK)
    return code;
  if (prep > 0 && (code = launch(e->prep, prep, 1, 256, &p, stream, "row-term")) != FA_OK) return code;
  if ((code = launch(e->main, kv_total + q_total, 1, 256, &p, stream, "backward")) != FA_OK) return code;
  if (sums > 0 && (code = launch(e->reduce, (sums + 255) / 256, 1, 256, &p, stream, "gradient sum")) != FA_OK) return code;
  return ok();
}

int kv4_append(const kv4_append_args* a, void* stream) {
  if (a == nullptr) return fail(FA_EINVAL, "null argument block");
  const kv4_cache* c = &a->cache;
  int code = check_cache(c);
  if (code != FA_OK) return code;
  if (a->rows < 0) return fail(FA_EINVAL, "invalid row count %d", a->rows);
  if (c->B == 0 || a->rows == 0) return ok();
  if ((code = check_tensor("k", a->k, a->k_stride, c->D, 8)) != FA_OK) return code;
  if ((code = check_tensor("v", a->v, a->v_stride, c->D, 8)) != FA_OK) return code;
  if ((a->k_values == nullptr) != (a->v_values == nullptr))
    return fail(FA_EINVAL, "k_values and v_values go together");
  if (a->k_values != nullptr) {
    if ((code = check_tensor("k_values", a->k_values, a->k_values_stride, c->D, 8)) != FA_OK) return code;
    if ((code = check_tensor("v_values", a->v_values, a->v_values_stride, c->D, 8)) != FA_OK) return code;
  }
  if (a->start == nullptr) return fail(FA_EINVAL, "null start pointer");
  const fa::Kv4KernelEntry* e = find_kv4(c->dtype, c->D);
  if (e == nullptr) return fail(FA_ENOTSUP, "4-bit cache kernels for dtype=%d D=%d are not built", c->dtype, c->D);
  fa::Kv4AppendParams p;
  std::memset(&p, 0, sizeof(p));
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.k_values = static_cast<uint16_t*>(a->k_values);
  p.v_values = static_cast<uint16_t*>(a->v_values);
  p.k_codes = c->k_codes;
  p.k_scales = c->k_scales;
  p.v_codes = c->v_codes;
  p.v_scales = c->v_scales;
  p.start = a->start;
  p.count = a->count;
  copy3(p.sk, a->k_stride);
  copy3(p.sv, a->v_stride);
  copy3(p.skv, a->k_values_stride);
  copy3(p.svv, a->v_values_stride);
  for (int i = 0; i < 2; ++i) {
    p.code_stride[i] = c->code_stride[i];
    p.scale_stride[i] = c->scale_stride[i];
  }
  p.B = c->B; p.Hkv = c->H_kv; p.D = c->D; p.rows = a->rows; p.capacity = c->capacity;
  const int64_t threads = (int64_t)c->B * c->H_kv * a->rows * (c->D / 8);
  if ((code = check_grid((threads + 255) / 256, 256, "cache append")) != FA_OK) return code;
  if ((code = launch(e->append, (threads + 255) / 256, 2, 256, &p, stream, "cache append")) != FA_OK) return code;
  return ok();
}

int64_t kv4_attend_workspace_bytes(int32_t B, int32_t H, int32_t M, int32_t D, int32_t splits) {
  if (splits <= 1 || B <= 0 || H <= 0 || M <= 0 || D <= 0) return 0;
  const int64_t rows = (int64_t)splits * B * H * M;
  return align256(rows * D * 4) + rows * 8;
}

int32_t kv4_attend_splits(int32_t B, int32_t H, int32_t H_kv, int32_t M, int32_t D, int32_t capacity) {
  const fa::Kv4KernelEntry* e = find_kv4(FA_DTYPE_F16, D);  // alike for both types
  if (e == nullptr || B <= 0 || H_kv <= 0 || H < H_kv || M <= 0 || capacity <= 0) return 1;
  const Kv4Kind k = kv4_kind(e, (int64_t)M * (H / H_kv));
  const int64_t blocks = (int64_t)B * H_kv * k.row_blocks, room = 256LL * e->per_cu[k.kind];
  // as many as the chip (256 CUs) holds at once, none with less than 256 keys of a full cache
  int64_t splits = room / blocks;
  if (splits > capacity / 256) splits = capacity / 256;
  return splits < 1 ? 1 : (int32_t)(splits > 4096 ? 4096 : splits);
}

int kv4_attend(const kv4_attend_args* a, void* stream) {
  if (a == nullptr) return fail(FA_EINVAL, "null argument block");
  const kv4_cache* c = &a->cache;
  int code = check_cache(c);
  if (code != FA_OK) return code;
  if (a->H <= 0 || a->M < 0) return fail(FA_EINVAL, "invalid sizes H=%d M=%d", a->H, a->M);
  if (a->H % c->H_kv != 0)
    return fail(FA_EINVAL, "query heads H=%d must be a multiple of kv heads H_kv=%d", a->H, c->H_kv);
  if ((code = check_scale(a->sm_scale)) != FA_OK) return code;
  if (a->splits < 1 || a->splits > 4096) return fail(FA_EINVAL, "splits=%d is outside 1 .. 4096", a->splits);
  if (c->B == 0 || a->M == 0) return ok();
  if ((code = check_tensor("q", a->q, a->q_stride, c->D, 8)) != FA_OK) return code;
  if ((code = check_tensor("o", a->o, a->o_stride, c->D, 4)) != FA_OK) return code;
  if (a->start == nullptr) return fail(FA_EINVAL, "null start pointer");
  const int64_t rows = (int64_t)a->M * (a->H / c->H_kv);
  if (rows * c->H_kv > (0x7fffffffLL - 256) / c->B) return fail(FA_EINVAL, "too many query rows (%lld per kv head)",
                                                                  (long long)rows);
  const fa::Kv4KernelEntry* e = find_kv4(c->dtype, c->D);
  if (e == nullptr) return fail(FA_ENOTSUP, "4-bit cache kernels for dtype=%d D=%d are not built", c->dtype, c->D);
  fa::Kv4AttendParams p;
  std::memset(&p, 0, sizeof(p));
  const int64_t need = kv4_attend_workspace_bytes(c->B, a->H, a->M, c->D, a->splits);
  if (need > 0) {
    if (a->workspace == nullptr || a->workspace_bytes < need)
      return fail(FA_EWORKSPACE, "split workspace of %lld bytes needed, got %lld", (long long)need,
                  (long long)a->workspace_bytes);
    if (!aligned(a->workspace, 16)) return fail(FA_EINVAL, "workspace must be 16-byte aligned");
    p.ws_o = static_cast<float*>(a->workspace);
    p.ws_ml = reinterpret_cast<float*>(static_cast<char*>(a->workspace) +
                                       align256((int64_t)a->splits * c->B * a->H * a->M * c->D * 4));
  }
  p.q = static_cast<const uint16_t*>(a->q);
  p.o = static_cast<uint16_t*>(a->o);
  p.lse = a->lse;
  p.k_codes = c->k_codes;
  p.k_scales = c->k_scales;
  p.v_codes = c->v_codes;
  p.v_scales = c->v_scales;
  p.start = a->start;
  p.count = a->count;
  copy3(p.sq, a->q_stride);
  copy3(p.so, a->o_stride);
  copy3(p.sl, a->lse_stride);
  for (int i = 0; i < 2; ++i) {
    p.code_stride[i] = c->code_stride[i];
    p.scale_stride[i] = c->scale_stride[i];
  }
  p.B = c->B; p.H = a->H; p.Hkv = c->H_kv; p.M = a->M; p.group = a->H / c->H_kv; p.capacity = c->capacity;
  p.causal = a->causal ? 1 : 0;
  p.splits = a->splits;
  p.c = a->sm_scale * 1.4426950408889634f;
  const Kv4Kind k = kv4_kind(e, rows);
  p.row_blocks = (int32_t)k.row_blocks;
  const int64_t slots = (int64_t)c->B * a->splits;
  const int64_t blocks = k.row_blocks * slots * c->H_kv;
  if (slots > 0x7fffffffLL) return fail(FA_EINVAL, "too many splits (%lld)", (long long)slots);
  p.slots = (int32_t)slots;
  const int64_t all = (int64_t)c->B * a->H * a->M;
  const int how = a->splits > 32 ? 2 : (a->splits > 8 ? 1 : 0);
  const int64_t few = (all + 3) / 4 < 2048 ? (all + 3) / 4 : 2048;  // eight workgroups to a CU, a few rows to a wave
  const int64_t joins = a->splits > 1 ? (how > 0 ? all : few) : 0;
  const int joiners = how == 2 ? 1024 : 256;
  if ((code = check_grid(blocks, 256, "cache attention")) != FA_OK || (code = check_grid(joins, joiners, "cache merge")) != FA_OK)
    return code;
  if ((code = launch(e->attend[k.kind], blocks, 1, 256, &p, stream, "cache attention")) != FA_OK) return code;
  if (joins > 0 && (code = launch(e->merge[how], joins, 1, joiners, &p, stream, "cache merge")) != FA_OK) return code;
  return ok();
}

}  // extern "C"
