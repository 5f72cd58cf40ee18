// The pages of the 8-bit key/value cache (layout in include/fa_gfx950.h): giving them out, sharing, returning and
// moving them, all on the GPU, so that a serving loop needs no host round trip and can be captured into a HIP graph.
//
// The state is the page table and, for each page, the number of entries that name it. What an operation does is
// defined by that state alone (free pages are taken lowest first, in order of sequence and token), so results do not
// depend on the order in which the GPU runs the work: counts change by integer atomics only, and places in an order
// come from prefix sums. Deciding is the work of one workgroup (reserve, compact): it is some thousand integers and
// bound by the latency of a few dependent loads, where a second launch would cost more than more workgroups gain.
// Copying is a launch of its own, bound by memory.
#include "../fa_common.h"
#include "../fa_kernels.h"

namespace fa {

constexpr int kPlanThreads = 1024, kThreads = 256;

// Reads and writes of words that other lanes change with atomics: those act in L2, past this CU's cache.
__device__ inline int load_shared(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ inline void store_shared(int* p, int x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// A barrier behind which they, and what this workgroup has written to its workspace, can be read: all of it has reached
// L2, of which a workgroup sees one. (A device-wide fence would write L2 back: 2 us each.)
__device__ inline void sync_shared() {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
}

__device__ inline bool is_page(const Kv8Pages& c, int page) { return (uint32_t)page < (uint32_t)c.pages; }

// Sum of x over the workgroup's threads before this one; `total` over all. The workgroup is kPlanThreads.
__device__ inline uint32_t prefix_sum(uint32_t x, uint32_t& total, uint32_t* parts) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t end = x;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) {
    const uint32_t o = __shfl_up(end, k, 64);
    if (lane >= k) end += o;
  }
  __syncthreads();  // of the last use of parts
  if (lane == 63) parts[wave] = end;
  __syncthreads();
  constexpr int WAVES = kPlanThreads / 64;
  uint32_t all = lane < WAVES ? parts[lane] : 0;
#pragma unroll
  for (int k = 1; k < WAVES; k *= 2) {
    const uint32_t o = __shfl_up(all, k, 64);
    if (lane >= k) all += o;
  }
  total = __shfl(all, WAVES - 1, 64);
  return end - x + (wave > 0 ? __shfl(all, wave - 1, 64) : 0u);
}

// Kinds of item (an entry that a call is asked to make writable).
enum { kHeld = 0, kNew = 1, kCopy = 2 };

struct Item {
  int64_t at;  // of the entry in the table
  int entry;   // -1 if nothing is asked of it
  int kind;
};
__device__ inline Item item_of(const Kv8PageParams& p, int i) {
  const Kv8Pages& c = p.cache;
  const int b = i / p.span, s = i - b * p.span;
  int n = p.count != nullptr ? p.count[b] : p.rows;
  n = n < 0 ? 0 : (n > p.rows ? p.rows : n);
  const int64_t start = p.a[b];
  const int64_t low = start > 0 ? start : 0, high = start + n < p.capacity ? start + n : p.capacity;
  const int page_log2 = 5 + c.blocks_log2;
  const int64_t column = (low >> page_log2) + s;
  const bool active = high > low && column << page_log2 < high;  // so column < columns: high <= capacity
  Item x;
  x.at = (int64_t)b * c.columns + column;
  x.entry = active ? c.table[x.at] : -1;
  x.kind = !active ? kHeld : (!is_page(c, x.entry) ? kNew : (c.refs[x.entry] > 1 ? kCopy : kHeld));
  return x;
}

// Pages for tokens. Items are looked at in order, a run of them to a thread. An entry whose page has other holders is
// copied unless it is the last of them and all of them are items: marked by the largest item and the number of items of
// each page. Then the items that want a page are counted, as many free pages are found from the lowest on, and the k-th
// item takes the k-th page.
// HELD: items stay in registers, EACH to a thread, and the pages found in LDS (up to 8192 items); otherwise they are
// looked up again and kept in the workspace. One decode step of 32 sequences 5 us, the prompts of 32 sequences of 2-4k
// tokens 9, where the workspace form takes 8 and 18. Bound by five dependent loads and the barriers between them.
constexpr int kHeldItems = 8;
template <bool HELD>
__global__ __launch_bounds__(kPlanThreads) void kv8_reserve_kernel(Kv8PageParams p) {
  constexpr int EACH = HELD ? kHeldItems : 1;
  __shared__ uint32_t parts[kPlanThreads / 64];
  __shared__ int copies;
  __shared__ int pages[HELD ? kPlanThreads * EACH : 1];
  const Kv8Pages& c = p.cache;
  const int items = p.B * p.span, each = (items + kPlanThreads - 1) / kPlanThreads;
  const int i0 = (int)min((int64_t)threadIdx.x * each, (int64_t)items), i1 = min(i0 + each, items);
  int* last = p.mark;
  int* sharers = p.mark + c.pages;
  Item held[EACH];
  // f(item, its number) of the thread's items; the kind that f leaves is kept
  auto for_items = [&](auto f) {
    if constexpr (HELD) {
#pragma unroll
      for (int k = 0; k < EACH; ++k)
        if (i0 + k < i1) f(held[k], i0 + k);
    } else {
      for (int i = i0; i < i1; ++i) {
        Item x = item_of(p, i);
        x.kind = p.wants[i];
        f(x, i);
        p.wants[i] = x.kind;
      }
    }
  };
  uint32_t wanted = 0;
  bool shared = false;
  if (threadIdx.x == 0) copies = 0;
  if constexpr (HELD) {
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      held[k] = {0, -1, kHeld};
      if (i0 + k < i1) held[k] = item_of(p, i0 + k);
    }
  } else {
    for (int i = i0; i < i1; ++i) p.wants[i] = item_of(p, i).kind;
  }
  for_items([&](Item& x, int) {
    wanted += x.kind == kNew;
    if (x.kind == kCopy) {
      shared = true;
      store_shared(last + x.entry, -1);
      store_shared(sharers + x.entry, 0);
    }
  });
  if (__syncthreads_or(shared)) {
    sync_shared();
    if (shared)
      for_items([&](Item& x, int i) {
        if (x.kind == kCopy) {
          atomicMax(last + x.entry, i);
          atomicAdd(sharers + x.entry, 1);
        }
      });
    sync_shared();
    if (shared)
      for_items([&](Item& x, int i) {
        if (x.kind == kCopy) {
          if (load_shared(last + x.entry) == i && load_shared(sharers + x.entry) == c.refs[x.entry]) x.kind = kHeld;
          else ++wanted;
        }
      });
    __syncthreads();  // refs are read above and changed below
  }
  uint32_t total;
  uint32_t rank = prefix_sum(wanted, total, parts);
  uint32_t found = 0;
  constexpr int RUN = 8;  // pages to a thread and step
  for (int64_t base = 0; base < c.pages && found < total; base += (int64_t)kPlanThreads * RUN) {
    const int64_t first = base + (int)threadIdx.x * RUN;
    uint32_t free = 0;  // a bit for each
    if (first + RUN <= c.pages) {
      int refs[RUN];
#pragma unroll
      for (int k = 0; k < RUN; ++k) refs[k] = c.refs[first + k];
#pragma unroll
      for (int k = 0; k < RUN; ++k) free |= (refs[k] == 0 ? 1u : 0u) << k;
    } else {
      for (int k = 0; k < RUN && first + k < c.pages; ++k) free |= (c.refs[first + k] == 0 ? 1u : 0u) << k;
    }
    uint32_t here;
    uint32_t at = found + prefix_sum((uint32_t)__popc(free), here, parts);
    for (; free != 0 && at < total; free &= free - 1, ++at) {
      const int page = (int)first + __builtin_ctz(free);
      if constexpr (HELD) pages[at] = page;
      else p.target[at] = page;
    }
    found += here;
  }
  const uint32_t given = found < total ? found : total;
  sync_shared();  // the k-th item that wants a page takes pages[k]; refs are read above and changed below
  if (wanted != 0)
    for_items([&](Item& x, int) {
      if (x.kind == kHeld) return;
      if (rank < given) {
        const int page = HELD ? pages[HELD ? rank : 0] : p.target[rank];
        c.table[x.at] = page;
        store_shared(c.refs + page, 1);
        if (x.kind == kCopy) {
          atomicSub(c.refs + x.entry, 1);
          const int k = atomicAdd(&copies, 1);
          p.source[2 * k] = x.entry;
          p.source[2 * k + 1] = page;
        }
      }
      ++rank;
    });
  __syncthreads();
  if (threadIdx.x == 0) {
    p.plan[0] = copies;
    p.result[0] = (int)(total - given);
  }
}

// A workgroup takes some columns of all sequences: every entry is read before one is written. 32 sequences of 32 columns
// 4.3 us: a launch and two loads, one behind the other, then the counts' atomics.
__global__ __launch_bounds__(kThreads) void kv8_fork_kernel(Kv8PageParams p) {
  __shared__ int old[kForkEntries];
  const Kv8Pages& c = p.cache;
  const int first = blockIdx.x * p.columns_each, n = min(p.columns_each, c.columns - first);
  for (int i = threadIdx.x; i < p.B * n; i += kThreads) old[i] = c.table[(int64_t)(i / n) * c.columns + first + i % n];
  __syncthreads();
  for (int i = threadIdx.x; i < p.B * n; i += kThreads) {
    const int b = i / n, parent = p.a[b];
    const int was = old[i], is = (uint32_t)parent < (uint32_t)p.B ? old[parent * n + i % n] : -1;
    if (is == was) continue;
    c.table[(int64_t)b * c.columns + first + i % n] = is;
    if (is_page(c, was)) atomicSub(c.refs + was, 1);
    if (is_page(c, is)) atomicAdd(c.refs + is, 1);
  }
}

// Every entry of the table, a lane to each; 32 x 128 of them 2.8 us, a launch.
__global__ __launch_bounds__(kThreads) void kv8_truncate_kernel(Kv8PageParams p) {
  const Kv8Pages& c = p.cache;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= (int64_t)p.B * c.columns) return;
  const int64_t column = i % c.columns;
  if (column << (5 + c.blocks_log2) < p.a[i / c.columns]) return;
  const int page = c.table[i];
  if (page == -1) return;
  c.table[i] = -1;
  if (is_page(c, page)) atomicSub(c.refs + page, 1);
}

// Which pages move where: the k-th used page at or behind the number of used pages goes to the k-th free one before it.
// p.mark: the new number of each page from there on. 2048 pages: 4.8 us, as reserve.
__global__ __launch_bounds__(kPlanThreads) void kv8_compact_kernel(Kv8PageParams p) {
  __shared__ uint32_t parts[kPlanThreads / 64];
  const Kv8Pages& c = p.cache;
  constexpr int RUN = 8;
  auto used_of = [&](int64_t first) {  // a bit for each of RUN pages
    uint32_t used = 0;
    if (first + RUN <= c.pages) {
      int refs[RUN];
#pragma unroll
      for (int k = 0; k < RUN; ++k) refs[k] = c.refs[first + k];
#pragma unroll
      for (int k = 0; k < RUN; ++k) used |= (refs[k] != 0 ? 1u : 0u) << k;
    } else {
      for (int k = 0; k < RUN && first + k < c.pages; ++k) used |= (c.refs[first + k] != 0 ? 1u : 0u) << k;
    }
    return used;
  };
  uint32_t mine = 0, live, used_now = 0;
  for (int64_t base = 0; base < c.pages; base += (int64_t)kPlanThreads * RUN) {
    used_now = used_of(base + (int)threadIdx.x * RUN);
    mine += (uint32_t)__popc(used_now);
  }
  prefix_sum(mine, live, parts);
  uint32_t moved = 0, holes = 0;
  for (int64_t base = 0; base < c.pages; base += (int64_t)kPlanThreads * RUN) {
    const int64_t first = base + (int)threadIdx.x * RUN;
    const uint32_t used = c.pages <= kPlanThreads * RUN ? used_now : used_of(first);  // one step: it is known
    const int inside = first >= c.pages ? 0 : (int)(c.pages - first < RUN ? c.pages - first : RUN);
    const int low = first >= live ? 0 : (int)(live - first < inside ? live - first : inside);  // pages before `live`
    const uint32_t low_bits = (1u << low) - 1, all_bits = (1u << inside) - 1;
    uint32_t hole = ~used & low_bits, move = used & all_bits & ~low_bits;
    // both counts in one sum: a step has kPlanThreads * RUN = 8192 pages
    uint32_t here;
    const uint32_t before = prefix_sum((uint32_t)__popc(move) | (uint32_t)__popc(hole) << 16, here, parts);
    uint32_t at = holes + (before >> 16);
    for (; hole != 0; hole &= hole - 1) p.target[at++] = (int)first + __builtin_ctz(hole);
    at = moved + (before & 0xffffu);
    for (int k = low; k < inside; ++k) {
      if (move >> k & 1u) p.source[at++] = (int)first + k;
      else p.mark[first + k] = (int)first + k;
    }
    moved += here & 0xffffu;
    holes += here >> 16;
  }
  sync_shared();  // of refs too: read above, changed below
  for (uint32_t k = threadIdx.x; k < moved; k += kPlanThreads) {
    const int from = p.source[k], to = p.target[k];
    p.mark[from] = to;
    c.refs[to] = c.refs[from];
    c.refs[from] = 0;
  }
  if (threadIdx.x == 0) {
    p.plan[0] = (int)moved;
    p.plan[1] = (int)live;
    p.result[0] = (int)live;
  }
}

// Copies the planned pages, all layers, and (MAP) writes the table's new entries. The host does not know how many there
// are: workgroups take slices in turn until there is none left. 269 MB read and as much written 90 us right after a call
// that read them (6.0 TB/s; a large copy has 4.8), 16 pages of 32 layers (67 MB and as much) 26 us, 5.2 TB/s.
template <bool MAP>
__global__ __launch_bounds__(kThreads) void kv8_move_kernel(Kv8PageParams p) {
  const Kv8Pages& c = p.cache;
  const int copies = p.plan[0];
  if constexpr (MAP) {
    const int live = p.plan[1];
    if (copies > 0)
      for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < (int64_t)p.B * c.columns; i += (int64_t)gridDim.x * kThreads) {
        const int page = c.table[i];
        if (is_page(c, page) && page >= live) c.table[i] = p.mark[page];
      }
  }
  const int64_t all = (int64_t)copies * p.layers * p.slices;
  for (int64_t unit = blockIdx.x; unit < all; unit += gridDim.x) {
    const int slice = (int)(unit % p.slices);
    const int64_t rest = unit / p.slices;
    const int layer = (int)(rest % p.layers);
    const int64_t k = rest / p.layers;
    const int from = MAP ? p.source[k] : p.source[2 * k], to = MAP ? p.target[k] : p.source[2 * k + 1];
    const uint8_t* src = c.data + layer * c.layer_stride + from * c.page_stride;
    uint8_t* dst = c.data + layer * c.layer_stride + to * c.page_stride;
    const int64_t end = min((slice + 1) * p.slice_bytes, p.page_bytes);
    constexpr int DEPTH = 4, STEP = kThreads * 16;
    for (int64_t at = slice * p.slice_bytes + threadIdx.x * 16; at < end; at += DEPTH * STEP) {
      u32x4 x[DEPTH];
#pragma unroll
      for (int j = 0; j < DEPTH; ++j)
        if (at + j * STEP < end) x[j] = *reinterpret_cast<const u32x4*>(src + at + j * STEP);
#pragma unroll
      for (int j = 0; j < DEPTH; ++j)
        // past the caches: the copies are read much later (134 MB of copied pages 42 -> 36 us with the rest of the call)
        if (at + j * STEP < end) __builtin_nontemporal_store(x[j], reinterpret_cast<u32x4*>(dst + at + j * STEP));
    }
  }
}

Kv8PageKernels kv8_page_kernels() {
  return {{(const void*)&kv8_reserve_kernel<false>, (const void*)&kv8_reserve_kernel<true>}, kHeldItems * kPlanThreads,
           (const void*)&kv8_fork_kernel,       (const void*)&kv8_truncate_kernel,
          (const void*)&kv8_compact_kernel,   (const void*)&kv8_move_kernel<false>, (const void*)&kv8_move_kernel<true>,
          kPlanThreads, kThreads};
}

}  // namespace fa
