// What attention over the 4-bit and the 8-bit cache have in common: the running maximum, how the sequences' keys are
// cut into splits, and the join of the splits. A parameter block `Params` has Kv4AttendParams' fields of those names.
#pragma once

#include "fa_common.h"
#include "../../include/fa_gfx950.h"

namespace fa {

// log2 of what P is scaled by on its way to the type; fp16: weights down to 2^-29 keep all their bits.
template <typename Tag>
__device__ constexpr float weight_bias();
template <>
__device__ constexpr float weight_bias<f16_t>() { return 15.f; }
template <>
__device__ constexpr float weight_bias<bf16_t>() { return 0.f; }

constexpr int kMaxCapacity = KV4_MAX_CAPACITY;
static_assert(KV8_MAX_CAPACITY == KV4_MAX_CAPACITY, "one bound for both caches");

// The larger of two scores, NaN if one is: one instruction, where fmaxf has to quiet each operand first.
__device__ inline float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Of a row's scores, over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ inline float row_max(float x) {
  uint32_t u = __float_as_uint(x);
  const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  u = __float_as_uint(larger(__uint_as_float(h[0]), __uint_as_float(h[1])));
  const auto q = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return larger(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

__device__ inline float scale_of(uint32_t e) { return __uint_as_float(e << 23); }

// Keys of sequence b that its rows may see.
__device__ inline int visible_keys(const int32_t* start, const int32_t* count, int b, int M, int capacity) {
  int n = count != nullptr ? count[b] : M;
  n = n < 0 ? 0 : (n > M ? M : n);
  const int64_t end = n == 0 ? 0 : (int64_t)start[b] + n;
  return end <= 0 ? 0 : (end > capacity ? capacity : (int)end);
}

// How the sequences' 32-key tiles are cut into splits: `per` tiles each, the fewest (but kMinTiles) that make at
// most B * splits splits of all sequences together, so that sequences of unequal lengths keep the workgroups
// equally long, and no more of them than the chip was said to hold: 800 where 768 fit took twice the time of
// 752. A split has a slot: sequence b's are those from its predecessors' number on. Each wave works this out
// from the lengths (64 sequences at a time, one to a lane).
constexpr int kMinTiles = 8;
constexpr int kAllTiles = kMaxCapacity / 32;  // of the largest cache: the share where nothing is split
static_assert(kMaxCapacity % 32 == 0 && (uint64_t)kAllTiles * 64 <= 0xffffffffu,
              "64 sequences of whole tiles are summed in 32 bits");

struct Split {
  int b, index;     // sequence, and which of its splits (b < 0: a slot that no split has)
  int first, used;  // the sequence's first slot and number of splits
  int per;          // tiles of a split
};

// The split of a slot (slot >= 0), or of sequence b (slot < 0: only first, used and per are set).
template <typename Params>
__device__ inline Split find_split(const Params& p, int slot, int b) {
  Split s;
  if (p.splits == 1) {
    s.b = slot;
    s.index = 0;
    s.first = slot;
    s.used = 1;
    s.per = kAllTiles;
    return s;
  }
  const int lane = threadIdx.x & 63;
  int64_t all = 0;
  int tiles = 0;
  for (int c = 0; c < p.B; c += 64) {
    tiles = c + lane < p.B ? (visible_keys(p.start, p.count, c + lane, p.M, p.capacity) + 31) / 32 : 0;
    uint32_t sum = (uint32_t)tiles;  // of 64 sequences of at most 2^25 tiles each
    for (int k = 1; k < 64 && k < p.B; k *= 2) sum += (uint32_t)__shfl_xor((int)sum, k, 64);
    all += (uint32_t)__builtin_amdgcn_readfirstlane((int)sum);
  }
  const int64_t most = (int64_t)p.B * p.splits;
  int64_t per = (all + most - 1) / most;
  if (per < kMinTiles) per = kMinTiles;
  const int64_t safe = (all + most - p.B - 1) / (most - p.B);  // sum of ceil(t / per) < all / per + B
  if (p.B > 64) {
    per = per > safe ? per : safe;
  } else {
    while (per < safe) {  // a sixteenth longer at a time
      int n = (tiles + (int)per - 1) / (int)per;
      for (int k = 1; k < p.B; k *= 2) n += __shfl_xor(n, k, 64);
      if (__builtin_amdgcn_readfirstlane(n) <= most) break;
      per += (per + 15) / 16;
    }
  }
  s.per = (int)per;
  s.b = -1;
  s.index = s.first = s.used = 0;
  int base = 0;
  for (int c = 0; c < p.B; c += 64) {
    if (p.B > 64) tiles = c + lane < p.B ? (visible_keys(p.start, p.count, c + lane, p.M, p.capacity) + 31) / 32 : 0;
    const int n = (tiles + s.per - 1) / s.per;
    int end = n;  // of the lane's splits
    for (int k = 1; k < 64 && k < p.B; k *= 2) {
      const int o = __shfl_up(end, k, 64);
      if (lane >= k) end += o;
    }
    end += base;
    const uint64_t hit = __ballot(slot >= 0 ? slot < end : c + lane == b);
    if (hit != 0) {
      const int who = __builtin_ctzll(hit);
      s.b = c + who;
      s.used = __builtin_amdgcn_readlane(n, who);
      s.first = __builtin_amdgcn_readlane(end, who) - s.used;
      s.index = slot - s.first;
      return s;
    }
    base = __builtin_amdgcn_readlane(end, 63);  // another 64 sequences follow, so all steps were made
  }
  return s;
}

// Joins the splits of a row: weights exp2((m_s - m) unit) of the unnormalised partial sums; the maxima m_s are scores with
// `unit` log2 units to one (the difference comes first: far from zero a product with the unit would be rounded to more than
// scores may differ by), or in log2 units with 1. WPR waves take a row: one
// where rows are many and splits few, four or sixteen the other way round (single tokens over long caches). D / 4 lanes read one
// split's row, so a wave has 256 / D of them in flight at once, times the unrolling.
template <typename Tag, int D, int WPR, typename Params>
__device__ inline void merge_splits(const Params& p, float unit) {
  constexpr int LPS = D / 4, AT_ONCE = WPR * 64 / LPS;
  __shared__ floatx4 part_o[WPR][LPS];
  __shared__ float part_ml[WPR][2];
  const int lane = threadIdx.x & 63, wave = WPR > 1 ? threadIdx.x >> 6 : 0;
  const uint32_t rows = (uint32_t)p.B * p.H * p.M;
  const uint32_t first = WPR > 1 ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 6);
  Split part;
  int of = -1;  // the sequence that `part` is of
  // a workgroup per row, or so many waves that each takes a few rows
  for (uint32_t row = __builtin_amdgcn_readfirstlane(first); row < rows; row += WPR > 1 ? rows : gridDim.x * 4) {
    const uint32_t bh = row / (uint32_t)p.M;
    const int i = (int)(row % (uint32_t)p.M), h = (int)(bh % (uint32_t)p.H), b = (int)(bh / (uint32_t)p.H);
    if (b != of) part = find_split(p, -1, of = b);
    const int64_t stride = (int64_t)p.H * p.M;  // rows of a slot
    const int64_t at = part.first * stride + (int64_t)h * p.M + i;
    const int mine = wave * (64 / LPS) + lane / LPS, c4 = lane % LPS;
    float m = FA_NEG_INF, sum = 0.f;
    floatx4 o = (floatx4){0.f, 0.f, 0.f, 0.f};
    for (int s = mine; s < part.used; s += AT_ONCE) m = fmaxf(m, p.ws_ml[2 * (at + s * stride)]);
    const float base = m == FA_NEG_INF ? 0.f : m;
#pragma unroll 4
    for (int s = mine; s < part.used; s += AT_ONCE) {
      const int64_t w = at + s * stride;
      const float f = fast_exp2((p.ws_ml[2 * w] - base) * unit);
      const floatx4 x = *reinterpret_cast<const floatx4*>(p.ws_o + w * D + 4 * c4);
      sum = fmaf(f, p.ws_ml[2 * w + 1], sum);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = fmaf(f, x[j], o[j]);
    }
#pragma unroll
    for (int k = LPS; k < 64; k *= 2) {  // the wave's lane groups
      const float mo = __shfl_xor(m, k, 64), so = __shfl_xor(sum, k, 64);
      const float top = fmaxf(m, mo), ref = top == FA_NEG_INF ? 0.f : top;
      const float f = fast_exp2((m - ref) * unit), fo = fast_exp2((mo - ref) * unit);
      sum = f * sum + fo * so;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = f * o[j] + fo * __shfl_xor(o[j], k, 64);
      m = top;
    }
    if constexpr (WPR > 1) {
      if (lane < LPS) part_o[wave][c4] = o;
      if (lane == 0) {
        part_ml[wave][0] = m;
        part_ml[wave][1] = sum;
      }
      __syncthreads();
      if (threadIdx.x >= LPS) return;  // there is no other row
      float top = FA_NEG_INF;
#pragma unroll
      for (int w = 0; w < WPR; ++w) top = fmaxf(top, part_ml[w][0]);
      const float ref = top == FA_NEG_INF ? 0.f : top;
      sum = 0.f;
      o = (floatx4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WPR; ++w) {
        const float f = fast_exp2((part_ml[w][0] - ref) * unit);
        sum = fmaf(f, part_ml[w][1], sum);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(f, part_o[w][c4][j], o[j]);
      }
      m = top;
    }
    if (lane >= LPS) continue;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<u32x2*>(p.o + b * p.so[0] + h * p.so[1] + i * p.so[2] + 4 * c4) =
        (u32x2){DT<Tag>::pack2(o[0] * inv, o[1] * inv), DT<Tag>::pack2(o[2] * inv, o[3] * inv)};
    if (c4 == 0 && p.lse != nullptr)
      p.lse[b * p.sl[0] + h * p.sl[1] + i * p.sl[2]] =
          sum == 0.f ? FA_NEG_INF : (m * unit + __builtin_amdgcn_logf(sum) - weight_bias<Tag>()) * 0.6931471805599453f;
  }
}

}  // namespace fa
