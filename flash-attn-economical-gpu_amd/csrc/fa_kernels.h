// Host-visible kernel parameter blocks and registries shared between the kernel translation units
// and the C ABI (fa_abi.hip).
#pragma once

#include <stdint.h>

namespace fa {

// One attention-forward launch. Pointers are device pointers; strides are in elements.
struct FwdParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  float* lse;     // nullable: fp32 [B,H,M] natural-log sum-exp of the scaled logits
  float* ws_o;    // split partials [splits][B*H][M][D] fp32 (SPLIT kernels only)
  float* ws_lse;  // split partial lse [splits][B*H][M] fp32 (SPLIT kernels only)
  int64_t sq0, sq1, sq2;
  int64_t sk0, sk1, sk2;
  int64_t sv0, sv1, sv2;
  int64_t so0, so1, so2;
  int64_t sl0, sl1, sl2;
  int32_t B, H, Hkv, M, N;
  int32_t group;            // H / Hkv
  int32_t pack;             // 1, or group: the query heads of a kv head share one row space
                            // (row r = head offset r / M, position r % M); grid over (b, kv head)
  float c;                  // sm_scale * log2(e): exp(x*sm_scale) == exp2(x*c)
  float sm_scale;
  int32_t causal;
  int32_t splits;           // KV splits (1 when not splitting)
  int32_t tiles_per_split;  // KV tiles (of block_n rows) per split
  int32_t m_blocks;         // ceil(M / block_m)
  int32_t total_blocks;     // m_blocks * B * H * splits
  int32_t grid;             // workgroups launched (the persistent kernel's; total_blocks otherwise)
};

struct MergeParams {
  const float* ws_o;
  const float* ws_lse;
  uint16_t* o;
  float* lse;
  int64_t so0, so1, so2;
  int64_t sl0, sl1, sl2;
  int32_t B, H, M, splits;
  int32_t waves_per_row;  // 1, 2 or 4: the waves of a workgroup that share one row's splits
};

typedef void (*FwdKernelFn)(FwdParams);
typedef void (*MergeKernelFn)(MergeParams);

struct FaKernelEntry {
  int32_t stages;  // 1 = basic, 2 = double-buffered K/V LDS (optimized), 3-5 = LDS-DMA pipelines
                   // (32x32x16 MFMAs), 6-10 = 16x16x32 MFMA kernels: 6 lean, 7 software-pipelined,
                   // 8 ping-pong, 9 persistent ping-pong, 10 key groups (fa_fwd16.hip)
  int32_t dtype;   // FA_DTYPE_*
  int32_t D;
  int32_t waves;
  int32_t rows_per_wave;
  int32_t block_n;
  int32_t split;   // writes fp32 partials for the LSE merge
  const void* fn;
  const char* symbol;  // mangled kernel name (the key of the build's resource table)
  // The basic kernels of fa_fwd16.hip run the body of another stages number: its launch rules apply
  // (addressing limits, grid), and its KV tile may be smaller than the block_n the tile names.
  int32_t body_stages = 0;
  int32_t body_block_n = 0;
  int32_t pipeline() const { return body_stages ? body_stages : stages; }
  int32_t kv_tile() const { return body_block_n ? body_block_n : block_n; }
};

struct FaMergeEntry {
  int32_t dtype;
  int32_t D;
  const void* fn;
};

// One attention-backward launch (row-term kernel, then dK/dV and dQ blocks in one grid). Strides
// are in elements: batch, head, row.
struct BwdParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* o;
  const uint16_t* dout;
  const float* lse;
  const float* dlse;  // nullable
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  int64_t sq[3], sk[3], sv[3], so[3], sdo[3], sl[3], sdl[3], sdq[3], sdk[3], sdv[3];
  float* nd;     // workspace: two fp32 terms per query row, in groups of 32 rows
  float* bound;  // workspace: block maxima behind fp16's dS scale
  float* ws_dk;  // workspace: partial gradients [kv_splits][B * Hkv][N][D] (kv_splits > 1)
  float* ws_dv;
  float* ws_dq;  // workspace: partial gradients [q_splits][B * H][M][D] (q_splits > 1)
  int32_t B, H, Hkv, M, N, group;
  int32_t row_groups;   // 32-row groups of a head's row terms
  int32_t prep_blocks;  // row-term blocks of a query head
  int32_t vblocks;      // V-norm blocks of a kv head (fp16; 0 otherwise)
  int32_t nblocks, mblocks;   // dK/dV blocks of a kv head, dQ blocks of a query head
  int32_t kv_splits, q_splits;  // workgroups that share a block's steps
  int32_t kv_total, q_total;    // workgroups of each kind
  int32_t causal;
  float c;      // scale * log2(e)
  float scale;
};

struct BwdKernelEntry {
  int32_t dtype;
  int32_t D;
  const void* prep;
  const void* main;
  const void* reduce;
  int32_t block;      // keys (dK/dV) and query rows (dQ) of a workgroup
  int32_t prep_rows;  // rows of a row-term block
  int32_t per_cu;     // workgroups that the split rule counts on per CU (at D = 64 three fit where two are counted)
};

const BwdKernelEntry* fa_bwd_registry(int* count);

// The 4-bit cache (kv4.hip). Code and scale strides are in bytes: batch, head; cached rows are dense.
struct Kv4AppendParams {
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* k_values;  // nullable (both): what the appended rows now stand for
  uint16_t* v_values;
  uint8_t* k_codes;
  uint8_t* k_scales;
  uint8_t* v_codes;
  uint8_t* v_scales;
  const int32_t* start;
  const int32_t* count;  // nullable: all rows
  int64_t sk[3], sv[3], skv[3], svv[3];
  int64_t code_stride[2], scale_stride[2];
  int32_t B, Hkv, D, rows, capacity;
};

struct Kv4AttendParams {
  const uint16_t* q;
  uint16_t* o;
  float* lse;  // nullable
  const uint8_t* k_codes;
  const uint8_t* k_scales;
  const uint8_t* v_codes;
  const uint8_t* v_scales;
  const int32_t* start;
  const int32_t* count;  // nullable: all rows
  float* ws_o;           // splits > 1: unnormalised partial sums [slots][H][M][D]
  float* ws_ml;          // splits > 1: their row maximum (log2 units) and sum [slots][H][M][2]
  int64_t sq[3], so[3], sl[3];
  int64_t code_stride[2], scale_stride[2];
  int32_t B, H, Hkv, M, group, capacity;
  int32_t causal, splits;
  int32_t slots;  // splits that all sequences may have together: B * splits
  int32_t row_blocks;
  float c;  // scale * log2(e)
};

struct Kv4KernelEntry {
  int32_t dtype;
  int32_t D;
  const void* append;
  const void* merge[3];   // one, four and sixteen waves to a row
  const void* attend[3];  // 16 rows shared by a workgroup's waves, 32 rows shared, chunks of a prompt
  int32_t per_cu[3];      // workgroups of each that the split rule counts on per CU (chunks at D = 64: three fit)
  int32_t chunk_rows;     // query rows of a workgroup of the last
};

const Kv4KernelEntry* kv4_registry(int* count);

// The paged 8-bit cache (kv8.hip, kv8_pages.hip). Strides of it are in bytes. The page layout is that of kv8_cache in
// include/fa_gfx950.h.
struct Kv8Pages {
  uint8_t* data;  // of one layer (append, attention), or of all
  int32_t* table;
  int32_t* refs;
  int64_t layer_stride, page_stride;
  int64_t scales_at;    // bytes of a page's codes
  int32_t pages, columns;
  int32_t blocks_log2;  // 32-token blocks of a page
};

struct Kv8AppendParams {
  Kv8Pages cache;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* k_values;  // nullable (both): what the appended rows now stand for
  uint16_t* v_values;
  const int32_t* start;
  const int32_t* count;  // nullable: all rows
  int64_t sk[3], sv[3], skv[3], svv[3];
  int32_t B, Hkv, rows, capacity;
  int32_t blocks;  // blocks that `rows` tokens may lie in
};

// n / d by a multiplication: (high half of n * multiplier + n) >> shift, for n < 2^31.
struct Divisor {
  uint32_t multiplier;
  int32_t shift;
  static Divisor of(int64_t d) {
    Divisor x = {0, 0};
    while ((1LL << x.shift) < d) ++x.shift;
    x.multiplier = (uint32_t)(((1ULL << 32) * (uint64_t)((1LL << x.shift) - d)) / (uint64_t)d + 1);
    return x;
  }
};

struct Kv8AttendParams {
  Kv8Pages cache;
  const uint16_t* q;
  uint16_t* o;
  float* lse;  // nullable
  const int32_t* start;
  const int32_t* count;  // nullable: all rows
  float* ws_o;           // splits > 1: unnormalised partial sums [slots][H][M][D]
  float* ws_ml;          // splits > 1: their row maximum (a score; chunks: the reference) and sum [slots][H][M][2]
  int32_t* parts;        // chunks, splits > 1: first workgroup and number of parts [Hkv][B][row_blocks][2]
  int64_t sq[3], so[3], sl[3];
  int32_t B, H, Hkv, M, group, capacity;
  int32_t causal, splits;
  int32_t slots;  // splits that all sequences may have together: B * splits (chunks: heads of all sequences)
  int32_t row_blocks;
  Divisor by_group, by_blocks, by_slots;
  float c;  // scale * log2(e)
};

struct Kv8KernelEntry {
  int32_t dtype;
  int32_t D;
  const void* append;
  const void* merge[3];   // one, four and sixteen waves to a row
  const void* attend[3];  // 16 rows shared by a workgroup's waves, 32 rows shared, chunks of a prompt
  const void* join;       // of the last one's parts
  int32_t per_cu[3];      // workgroups of each that the split rule counts on per CU
  int32_t chunk_rows;     // query rows of a workgroup of the last
  int32_t join_rows;      // rows of a joining workgroup
};

const Kv8KernelEntry* kv8_registry(int* count);

struct Kv8PageParams {
  Kv8Pages cache;
  const int32_t* a;      // start, parent or length
  const int32_t* count;  // nullable: all rows
  int32_t* result;       // missing or used pages
  int32_t* plan;         // workspace: number of copies, pages in use
  int32_t* source;       // workspace: pages to be copied, and where to
  int32_t* target;
  int32_t* mark;         // workspace, by page: last sharer and number of sharers (reserve), new page (compact)
  int32_t* wants;        // workspace, by item (reserve)
  int32_t B, rows, capacity, layers;
  int32_t span;            // entries that `rows` tokens may lie in
  int32_t columns_each;    // columns of the table that a workgroup takes (fork)
  int32_t slices;          // parts of a page that are copied by themselves
  int64_t slice_bytes, page_bytes;
};

// Kernels of the page operations, and the threads of a workgroup of each.
struct Kv8PageKernels {
  const void* reserve[2];  // items in the workspace; up to held_items of them in registers
  int32_t held_items;
  const void* fork;
  const void* truncate;
  const void* compact;
  const void* copy;  // of what reserve planned
  const void* move;  // of what compact planned
  int32_t plan_threads, threads;
};

constexpr int kForkEntries = 16384;  // entries of the table that a workgroup of fork holds in LDS (KV8_MAX_FORK)

Kv8PageKernels kv8_page_kernels();

// The last error of the calling thread (fa_last_error), shared by the files that implement the C ABI.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int ok();

const FaKernelEntry* fa_fwd_registry(int* count);
const FaKernelEntry* fa_fwd16_registry(int* count);
const FaMergeEntry* fa_merge_registry(int* count);

struct GemmParams {
  const uint16_t* a;
  const uint16_t* b;
  uint16_t* c;
  int32_t M, N, K;
  int64_t lda, ldb, ldc;
  int32_t group_m;
  int32_t tiles_m, tiles_n;
  int32_t region_m;  // 0: flat grouped order; else XCD regions in region_m rows x (8 / region_m) columns
  int32_t grid;      // workgroups launched (the persistent kernel walks tiles with this stride)
  // split K over the grid (gemm_f16_part_kernel, gemm_f16_reduce_kernel)
  float* ws;                // fp32 partial products [ksplits][M][N]
  int32_t ksplits;
  int32_t slabs_per_split;  // K slabs (of block_k) per split
};

struct GemmKernelEntry {
  int32_t block_m, block_n, block_k, waves;
  const void* fn;          // default slab ring (as deep as fits in 128 KiB, up to 4)
  const void* fn_shallow;  // shallow ring for short K (nullptr when it would be the same)
  const char* symbol;      // mangled name of `fn`
  const void* fn_persist;  // persistent short-K kernel (nullptr when not built for the tile)
  const void* fn_part = nullptr;  // split-K kernel (nullptr when not built for the tile)
};

// K slabs up to which a tile's shallow-ring kernel is launched (more workgroups per CU beat a
// deeper prefetch when the whole K loop is this short).
constexpr int kGemmShallowMaxSlabs = 8;
// K slabs for which a tile's persistent kernel is launched (when built and the shape divides into
// whole tiles): at least the slab steps over which it stores a tile's C, and few enough that the C
// write is a large share of the time.
constexpr int kGemmPersistMinSlabs = 4;
constexpr int kGemmPersistMaxSlabs = 16;
// Waves the persistent kernel adds to the tile's compute waves to write C (one per SIMD).
constexpr int kGemmPersistStoreWaves = 4;

const GemmKernelEntry* gemm_registry(int* count);
const void* gemm_reduce_fn();

// Resources of one kernel as the compiler reported them (-Rpass-analysis=kernel-resource-usage).
// The table is generated by build_lib.py after the kernels are compiled and linked into the
// library (_build/kernel_resource_table.cpp).
struct KernelResourceRow {
  const char* symbol;
  int32_t vgprs, agprs, sgprs, lds_bytes, scratch_bytes, occupancy;
};
extern const KernelResourceRow kKernelResourceRows[];
extern const int kKernelResourceRowCount;

}  // namespace fa
