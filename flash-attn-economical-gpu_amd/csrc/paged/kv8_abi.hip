// C ABI of the paged 8-bit key/value cache (declared in include/fa_gfx950.h): argument validation and launches on the
// caller's stream.
#include <hip/hip_runtime.h>

#include <cstring>

#include "../fa_abi_checks.h"
#include "../fa_kernels.h"
#include "../../../include/fa_gfx950.h"

namespace {

using namespace fa::abi;
using fa::fail;
using fa::ok;

const fa::Kv8KernelEntry* find_kv8(int dtype, int D) {
  int n = 0;
  const fa::Kv8KernelEntry* e = fa::kv8_registry(&n);
  for (int i = 0; i < n; ++i)
    if (e[i].dtype == dtype && e[i].D == D) return &e[i];
  return nullptr;
}

int64_t codes_bytes(int64_t Hkv, int64_t page, int64_t D) { return 2 * Hkv * page * D; }

int check_buffers(const kv8_cache* c) {
  if (!c->data || !c->refs) return fail(FA_EINVAL, "null cache pointer");
  if (!aligned(c->data, 16) || c->page_stride % 16 || c->layer_stride % 16)
    return fail(FA_EINVAL, "cache data and its strides must be 16-byte aligned");
  if (c->pages > 1 && c->page_stride < kv8_page_bytes(c->H_kv, c->page, c->D))
    return fail(FA_EINVAL, "page stride %lld is under a page's %lld bytes", (long long)c->page_stride,
                (long long)kv8_page_bytes(c->H_kv, c->page, c->D));
  if (c->layers > 1) {  // whole layers behind each other, or a page's layers
    const __int128 page = kv8_page_bytes(c->H_kv, c->page, c->D);
    const __int128 layer = page + (c->pages > 1 ? (c->pages - 1) * (__int128)c->page_stride : 0);
    const __int128 stack = page + (c->layers - 1) * (__int128)c->layer_stride;
    if (c->layer_stride < layer && (c->layer_stride < page || c->page_stride < stack))
      return fail(FA_EINVAL, "layers %lld bytes apart overlap", (long long)c->layer_stride);
  }
  return FA_OK;
}

int check_cache(const kv8_cache* c) {
  const int code = check_type(c->dtype, c->D);
  if (code != FA_OK) return code;
  if (c->B < 0 || c->H_kv <= 0 || c->pages < 1 || c->columns < 0 || c->capacity < 0 || c->layers < 1)
    return fail(FA_EINVAL, "invalid cache sizes B=%d H_kv=%d pages=%d columns=%d capacity=%d layers=%d", c->B, c->H_kv, c->pages,
                c->columns, c->capacity, c->layers);
  if (c->page != 32 && c->page != 64 && c->page != 128 && c->page != 256)
    return fail(FA_ENOTSUP, "pages of %d tokens are not built (32, 64, 128, 256)", c->page);
  if (c->H_kv > (1 << 20)) return fail(FA_ENOTSUP, "H_kv=%d is beyond 2^20", c->H_kv);
  if (c->capacity > KV8_MAX_CAPACITY) return fail(FA_ENOTSUP, "cache capacity %d is beyond %d", c->capacity, KV8_MAX_CAPACITY);
  if (c->pages > KV8_MAX_CAPACITY) return fail(FA_ENOTSUP, "%d pages are beyond %d", c->pages, KV8_MAX_CAPACITY);
  if ((int64_t)c->columns * c->page < c->capacity)
    return fail(FA_EINVAL, "%d columns of %d tokens do not hold the capacity %d", c->columns, c->page, c->capacity);
  if ((int64_t)c->B * c->columns > (1 << 30)) return fail(FA_EINVAL, "page table too large (%d x %d)", c->B, c->columns);
  if (c->B == 0 || c->columns == 0) return FA_OK;  // no call but compact reads anything
  if (!c->table) return fail(FA_EINVAL, "null cache pointer");
  return check_buffers(c);
}

fa::Kv8Pages pages_of(const kv8_cache* c, int layer) {
  fa::Kv8Pages p;
  std::memset(&p, 0, sizeof(p));
  p.data = c->data + layer * c->layer_stride;
  p.table = c->table;
  p.refs = c->refs;
  p.layer_stride = c->layer_stride;
  p.page_stride = c->page_stride;
  p.scales_at = codes_bytes(c->H_kv, c->page, c->D);
  p.pages = c->pages;
  p.columns = c->columns;
  p.blocks_log2 = c->page == 32 ? 0 : (c->page == 64 ? 1 : (c->page == 128 ? 2 : 3));
  return p;
}

int check_layer(const kv8_cache* c, int layer) {
  if (layer < 0 || layer >= c->layers) return fail(FA_EINVAL, "layer %d of %d", layer, c->layers);
  return FA_OK;
}

// Which attention kernel takes a kv head's query rows: up to 32 the waves of a workgroup share them (and the cache is read
// once, or by two workgroups of 16 rows); more go chunk_rows to a workgroup.
struct Kind {
  int kind;
  int64_t row_blocks;
};
Kind kind_of(const fa::Kv8KernelEntry* e, int64_t rows) {
  Kind k;
  k.kind = rows <= 32 ? (rows <= 16 || e->attend[1] == nullptr ? 0 : 1) : 2;
  const int64_t block = k.kind == 2 ? e->chunk_rows : 16 << k.kind;
  k.row_blocks = (rows + block - 1) / block;
  return k;
}

// Partial sums of the splits: [slots][H][M] rows, or two row blocks of a workgroup (chunks).
struct AttendWorkspace {
  int64_t ml_at, parts_at, bytes;
};
AttendWorkspace attend_workspace(const fa::Kv8KernelEntry* e, int64_t B, int64_t H, int64_t Hkv, int64_t M, int64_t D,
                                 int64_t splits) {
  const Kind k = kind_of(e, M * (H / Hkv));
  const int64_t rows = k.kind == 2 ? 2 * splits * e->chunk_rows : splits * B * H * M;
  AttendWorkspace w;
  w.ml_at = align256(rows * D * 4);
  w.parts_at = w.bytes = w.ml_at + rows * 8;
  if (k.kind == 2) w.bytes += 8 * B * Hkv * k.row_blocks;
  return w;
}

int check_workspace(const void* workspace, int64_t bytes, int64_t need, const char* what) {
  if (need > 0 && (workspace == nullptr || bytes < need))
    return fail(FA_EWORKSPACE, "%s workspace of %lld bytes needed, got %lld", what, (long long)need, (long long)bytes);
  if (!aligned(workspace, 16)) return fail(FA_EINVAL, "workspace must be 16-byte aligned");
  return FA_OK;
}

int64_t span_of(const kv8_cache* c, int64_t rows) {  // columns that `rows` tokens may lie in
  const int64_t span = rows <= 0 ? 0 : (rows + c->page - 2) / c->page + 1;
  return span < c->columns ? span : c->columns;
}

int64_t align16(int64_t n) { return (n + 15) & ~(int64_t)15; }

// The page operations' workspace: numbers, pairs or sources, targets, a mark or two for each page, items.
struct PageWorkspace {
  int64_t source_at, target_at, mark_at, wants_at, bytes;
};
PageWorkspace reserve_workspace(const kv8_cache* c, int64_t rows) {
  const int64_t items = c->B * span_of(c, rows), most = items < c->pages ? items : c->pages;
  PageWorkspace w;
  w.source_at = 16;
  w.target_at = w.source_at + align16(8 * most);
  w.mark_at = w.target_at + align16(4 * most);
  w.wants_at = w.mark_at + align16(8 * (int64_t)c->pages);
  w.bytes = w.wants_at + align16(4 * items);
  return w;
}
PageWorkspace compact_workspace(const kv8_cache* c) {
  PageWorkspace w;
  w.source_at = 16;
  w.target_at = w.source_at + align16(4 * (int64_t)c->pages);
  w.mark_at = w.target_at + align16(4 * (int64_t)c->pages);
  w.wants_at = w.bytes = w.mark_at + align16(4 * (int64_t)c->pages);
  return w;
}

fa::Kv8PageParams page_params(const kv8_cache* c) {
  fa::Kv8PageParams p;
  std::memset(&p, 0, sizeof(p));
  p.cache = pages_of(c, 0);
  p.B = c->B;
  p.capacity = c->capacity;
  p.layers = c->layers;
  p.page_bytes = kv8_page_bytes(c->H_kv, c->page, c->D);
  // slices of about 16 KB: four loads of 16 bytes in flight for each of 256 lanes
  p.slices = (int32_t)(p.page_bytes >= 16384 ? p.page_bytes / 16384 : 1);
  p.slice_bytes = align16((p.page_bytes + p.slices - 1) / p.slices);
  return p;
}

void set_workspace(fa::Kv8PageParams* p, void* workspace, const PageWorkspace& w) {
  char* ws = static_cast<char*>(workspace);
  p->plan = reinterpret_cast<int32_t*>(ws);
  p->source = reinterpret_cast<int32_t*>(ws + w.source_at);
  p->target = reinterpret_cast<int32_t*>(ws + w.target_at);
  p->mark = reinterpret_cast<int32_t*>(ws + w.mark_at);
  p->wants = reinterpret_cast<int32_t*>(ws + w.wants_at);
}

// Workgroups that copy at most `copies` pages: as many as there may be slices, up to four times what the chip holds at
// once (with 2048 in all, 540 MB took 129 us where 8192 take 120: the last slices of a few were waited for).
int64_t copy_blocks(const fa::Kv8PageParams& p, int64_t copies) {
  const int64_t all = copies * p.layers * p.slices;
  return all < 1 ? 1 : (all < 8192 ? all : 8192);
}

}  // namespace

extern "C" {

int64_t kv8_page_bytes(int32_t H_kv, int32_t page, int32_t D) {
  if (H_kv <= 0 || page <= 0 || D <= 0) return 0;
  return (codes_bytes(H_kv, page, D) + 2 * (int64_t)H_kv * (page / 32) + 127) & ~(int64_t)127;
}

int kv8_append(const kv8_append_args* a, void* stream) {
  if (a == nullptr) return fail(FA_EINVAL, "null argument block");
  const kv8_cache* c = &a->cache;
  int code = check_cache(c);
  if (code != FA_OK || (code = check_layer(c, a->layer)) != FA_OK) return code;
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
  const fa::Kv8KernelEntry* e = find_kv8(c->dtype, c->D);
  if (e == nullptr) return fail(FA_ENOTSUP, "8-bit cache kernels for dtype=%d D=%d are not built", c->dtype, c->D);
  fa::Kv8AppendParams p;
  std::memset(&p, 0, sizeof(p));
  p.cache = pages_of(c, a->layer);
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.k_values = static_cast<uint16_t*>(a->k_values);
  p.v_values = static_cast<uint16_t*>(a->v_values);
  p.start = a->start;
  p.count = a->count;
  copy3(p.sk, a->k_stride);
  copy3(p.sv, a->v_stride);
  copy3(p.skv, a->k_values_stride);
  copy3(p.svv, a->v_values_stride);
  p.B = c->B; p.Hkv = c->H_kv; p.rows = a->rows; p.capacity = c->capacity;
  p.blocks = (int32_t)(((int64_t)a->rows + 30) / 32 + 1);
  const int64_t waves = (int64_t)c->B * c->H_kv * p.blocks;
  if ((code = check_grid((waves + 3) / 4, 256, "cache append")) != FA_OK) return code;
  if ((code = launch(e->append, (waves + 3) / 4, 2, 256, &p, stream, "cache append")) != FA_OK) return code;
  return ok();
}

int64_t kv8_attend_workspace_bytes(int32_t B, int32_t H, int32_t H_kv, int32_t M, int32_t D, int32_t splits) {
  const fa::Kv8KernelEntry* e = find_kv8(FA_DTYPE_F16, D);  // alike for both types
  if (e == nullptr || splits <= 1 || B <= 0 || H_kv <= 0 || H < H_kv || M <= 0) return 0;
  return attend_workspace(e, B, H, H_kv, M, D, splits).bytes;
}

int32_t kv8_attend_splits(int32_t B, int32_t H, int32_t H_kv, int32_t M, int32_t D, int32_t capacity) {
  const fa::Kv8KernelEntry* e = find_kv8(FA_DTYPE_F16, D);
  if (e == nullptr || B <= 0 || H_kv <= 0 || H < H_kv || M <= 0 || capacity <= 0) return 1;
  const Kind k = kind_of(e, (int64_t)M * (H / H_kv));
  const int64_t blocks = (int64_t)B * H_kv * k.row_blocks, room = 256LL * e->per_cu[k.kind];
  // as many as the chip (256 CUs) holds at once, none with less than 256 keys of a full cache
  if (k.kind == 2) {
    // Twice as many blocks as fit are given out whole, the longest first: nothing is left to join. Whole / shares, us: two
    // sequences' first 2048 rows (32/8 heads, 1024 blocks) 88 / 156, one sequence's first 4096 157 / 217; below that, 512 rows
    // against 32k keys (128 blocks) 736 / 293, 2 x 509 against 16k (224) 537 / 305, 100 rows of 8/2 heads against 4k (8) 133 / 30.
    // The number of blocks alone does not tell: blocks that fit at once and are short are faster whole too (first 512 rows
    // 20 / 35, first 2048 rows of one sequence 60 / 97, 1024 rows of 16/4 heads, D = 256, against 16k 670 / 693).
    if (blocks >= 2 * room) return 1;
    const int64_t most = blocks * ((capacity + 255) / 256);
    return (int32_t)(most < room ? most : room);
  }
  int64_t splits = room / blocks;
  if (splits > capacity / 256) splits = capacity / 256;
  return splits < 1 ? 1 : (int32_t)(splits > 4096 ? 4096 : splits);
}

int kv8_attend(const kv8_attend_args* a, void* stream) {
  if (a == nullptr) return fail(FA_EINVAL, "null argument block");
  const kv8_cache* c = &a->cache;
  int code = check_cache(c);
  if (code != FA_OK || (code = check_layer(c, a->layer)) != FA_OK) return code;
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
  if (rows * c->H_kv > (0x7fffffffLL - 256) / c->B)
    return fail(FA_EINVAL, "too many query rows (%lld per kv head)", (long long)rows);
  const fa::Kv8KernelEntry* e = find_kv8(c->dtype, c->D);
  if (e == nullptr) return fail(FA_ENOTSUP, "8-bit cache kernels for dtype=%d D=%d are not built", c->dtype, c->D);
  fa::Kv8AttendParams p;
  std::memset(&p, 0, sizeof(p));
  if (a->splits > 1) {
    const AttendWorkspace w = attend_workspace(e, c->B, a->H, c->H_kv, a->M, c->D, a->splits);
    if ((code = check_workspace(a->workspace, a->workspace_bytes, w.bytes, "split")) != FA_OK) return code;
    char* ws = static_cast<char*>(a->workspace);
    p.ws_o = reinterpret_cast<float*>(ws);
    p.ws_ml = reinterpret_cast<float*>(ws + w.ml_at);
    p.parts = reinterpret_cast<int32_t*>(ws + w.parts_at);
  }
  p.cache = pages_of(c, a->layer);
  p.q = static_cast<const uint16_t*>(a->q);
  p.o = static_cast<uint16_t*>(a->o);
  p.lse = a->lse;
  p.start = a->start;
  p.count = a->count;
  copy3(p.sq, a->q_stride);
  copy3(p.so, a->o_stride);
  copy3(p.sl, a->lse_stride);
  p.B = c->B; p.H = a->H; p.Hkv = c->H_kv; p.M = a->M; p.group = a->H / c->H_kv; p.capacity = c->capacity;
  p.causal = a->causal ? 1 : 0;
  p.splits = a->splits;
  p.c = a->sm_scale * 1.4426950408889634f;
  const Kind k = kind_of(e, rows);
  p.row_blocks = (int32_t)k.row_blocks;
  p.by_group = fa::Divisor::of(p.group);
  p.by_blocks = fa::Divisor::of(k.row_blocks);
  if (k.kind == 2) {
    const int64_t all = k.row_blocks * c->B * c->H_kv;
    p.slots = c->B * c->H_kv;
    p.by_slots = fa::Divisor::of(p.slots);
    const int64_t blocks = a->splits > 1 ? a->splits : all, joins = a->splits > 1 ? all * (e->chunk_rows / e->join_rows) : 0;
    if ((code = check_grid(blocks, 256, "cache attention")) != FA_OK || (code = check_grid(joins, 256, "cache join")) != FA_OK)
      return code;
    if ((code = launch(e->attend[2], blocks, 1, 256, &p, stream, "cache attention")) != FA_OK) return code;
    if (joins > 0 && (code = launch(e->join, joins, 1, 256, &p, stream, "cache join")) != FA_OK) return code;
    return ok();
  }
  const int64_t slots = (int64_t)c->B * a->splits;
  const int64_t blocks = k.row_blocks * slots * c->H_kv;
  if (slots > 0x7fffffffLL) return fail(FA_EINVAL, "too many splits (%lld)", (long long)slots);
  p.slots = (int32_t)slots;
  p.by_slots = fa::Divisor::of(slots);
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

int64_t kv8_reserve_workspace_bytes(const kv8_cache* cache, int32_t rows) {
  return cache == nullptr || check_cache(cache) != FA_OK ? 0 : reserve_workspace(cache, rows).bytes;
}

int kv8_reserve(const kv8_reserve_args* a, void* stream) {
  if (a == nullptr) return fail(FA_EINVAL, "null argument block");
  const kv8_cache* c = &a->cache;
  int code = check_cache(c);
  if (code != FA_OK) return code;
  if (a->rows < 0) return fail(FA_EINVAL, "invalid row count %d", a->rows);
  if (a->missing == nullptr) return fail(FA_EINVAL, "null missing pointer");
  const int64_t span = span_of(c, a->rows);
  if (c->B * span > 0 && a->start == nullptr) return fail(FA_EINVAL, "null start pointer");
  const PageWorkspace w = reserve_workspace(c, a->rows);
  if ((code = check_workspace(a->workspace, a->workspace_bytes, w.bytes, "reserve")) != FA_OK) return code;
  fa::Kv8PageParams p = page_params(c);
  set_workspace(&p, a->workspace, w);
  p.a = a->start;
  p.count = a->count;
  p.result = a->missing;
  p.rows = a->rows;
  p.span = (int32_t)span;
  const fa::Kv8PageKernels k = fa::kv8_page_kernels();
  const int64_t items = c->B * span;
  if ((code = launch(k.reserve[items <= k.held_items], 1, 1, k.plan_threads, &p, stream, "page reserve")) != FA_OK) return code;
  if (items > 0 && c->pages > 1 &&
      (code = launch(k.copy, copy_blocks(p, items < c->pages ? items : c->pages), 1, k.threads, &p, stream, "page copy")) != FA_OK)
    return code;
  return ok();
}

int kv8_fork(const kv8_cache* c, const int32_t* parent, void* stream) {
  if (c == nullptr) return fail(FA_EINVAL, "null argument block");
  int code = check_cache(c);
  if (code != FA_OK) return code;
  if (c->B > KV8_MAX_FORK) return fail(FA_ENOTSUP, "fork of %d sequences (%d at most)", c->B, KV8_MAX_FORK);
  if (c->B == 0 || c->columns == 0) return ok();
  if (parent == nullptr) return fail(FA_EINVAL, "null parent pointer");
  fa::Kv8PageParams p = page_params(c);
  p.a = parent;
  // 64 columns, 256 bytes of a row, where LDS holds them for all sequences
  static_assert(KV8_MAX_FORK <= fa::kForkEntries, "a column of all sequences fits");
  const int64_t fit = fa::kForkEntries / c->B;
  p.columns_each = (int32_t)(fit < 64 ? fit : 64);
  const fa::Kv8PageKernels k = fa::kv8_page_kernels();
  const int64_t blocks = (c->columns + p.columns_each - 1) / p.columns_each;
  if ((code = check_grid(blocks, k.threads, "page fork")) != FA_OK) return code;
  if ((code = launch(k.fork, blocks, 1, k.threads, &p, stream, "page fork")) != FA_OK) return code;
  return ok();
}

int kv8_truncate(const kv8_cache* c, const int32_t* length, void* stream) {
  if (c == nullptr) return fail(FA_EINVAL, "null argument block");
  int code = check_cache(c);
  if (code != FA_OK) return code;
  if (c->B == 0 || c->columns == 0) return ok();
  if (length == nullptr) return fail(FA_EINVAL, "null length pointer");
  fa::Kv8PageParams p = page_params(c);
  p.a = length;
  const fa::Kv8PageKernels k = fa::kv8_page_kernels();
  const int64_t blocks = ((int64_t)c->B * c->columns + k.threads - 1) / k.threads;
  if ((code = launch(k.truncate, blocks, 1, k.threads, &p, stream, "page truncate")) != FA_OK) return code;
  return ok();
}

int64_t kv8_compact_workspace_bytes(const kv8_cache* cache) {
  return cache == nullptr || check_cache(cache) != FA_OK ? 0 : compact_workspace(cache).bytes;
}

int kv8_compact(const kv8_compact_args* a, void* stream) {
  if (a == nullptr) return fail(FA_EINVAL, "null argument block");
  const kv8_cache* c = &a->cache;
  int code = check_cache(c);
  if (code != FA_OK) return code;
  if ((code = check_buffers(c)) != FA_OK) return code;
  if (a->used == nullptr) return fail(FA_EINVAL, "null used pointer");
  const PageWorkspace w = compact_workspace(c);
  if ((code = check_workspace(a->workspace, a->workspace_bytes, w.bytes, "compact")) != FA_OK) return code;
  fa::Kv8PageParams p = page_params(c);
  set_workspace(&p, a->workspace, w);
  p.result = a->used;
  const fa::Kv8PageKernels k = fa::kv8_page_kernels();
  if ((code = launch(k.compact, 1, 1, k.plan_threads, &p, stream, "page compact")) != FA_OK) return code;
  if (c->pages > 1 &&
      (code = launch(k.move, copy_blocks(p, c->pages / 2), 1, k.threads, &p, stream, "page move")) != FA_OK)
    return code;
  return ok();
}

}  // extern "C"
