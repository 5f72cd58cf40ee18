// Paged 8-bit key/value cache for gfx950: append of new rows, and attention over the cache.
//
// Format. 32 consecutive tokens of a kv head are a block: one scale byte e, standing for 2^(e - 127), and an e4m3
// code for each channel. gfx950 converts such codes to fp16 or bf16, scale included, two to an instruction
// (v_cvt_scalef32_pk_*_fp8), so the products stay 16-bit MFMAs on exact values. A floating code keeps its relative
// step whatever the scale, so one power of two for 32 rows costs nothing until a channel lies 2^14 below the block's
// largest value. Blocks never cross a page, and a tile of the attention kernels is one or two whole blocks.
#include <limits>
#include <type_traits>

#include "../fa_common.h"
#include "../fa_kernels.h"
#include "../kv_split.h"
#include "../../../include/fa_gfx950.h"

namespace fa {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef short shortx2 __attribute__((ext_vector_type(2)));
typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));

template <typename Tag>
struct Fp8;
template <>
struct Fp8<f16_t> {
  // Range of scale bytes: the smallest and largest values, 2^-9 and 448 times 2^(e - 127), are numbers of the type.
  static constexpr uint32_t kFloor = 112, kCeil = 134;
  static constexpr uint32_t kInfBits = 0x7c00u;
  static constexpr uint32_t kMaxBits = 0x7b00u;  // 448 * 2^7
  template <bool HIGH>
  __device__ static inline shortx2 encode(shortx2 old, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(old, __builtin_bit_cast(half2_t, pair), scale, HIGH);
  }
  template <bool HIGH>
  __device__ static inline uint32_t decode(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HIGH));
  }
};
template <>
struct Fp8<bf16_t> {
  static constexpr uint32_t kFloor = 10, kCeil = 246;
  static constexpr uint32_t kInfBits = 0x7f80u;
  static constexpr uint32_t kMaxBits = 0x7f60u;  // 448 * 2^119
  template <bool HIGH>
  __device__ static inline shortx2 encode(shortx2 old, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(old, __builtin_bit_cast(bf16x2_t, pair), scale, HIGH);
  }
  template <bool HIGH>
  __device__ static inline uint32_t decode(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
  }
};

// Scale of a cached byte: one past the largest that append writes would make infinities of codes.
template <typename Tag>
__device__ inline float block_scale(uint32_t e) {
  return scale_of(e < Fp8<Tag>::kCeil ? e : Fp8<Tag>::kCeil);
}

// Four codes (a dword) to 16-bit values, two to a dword.
template <typename Tag>
__device__ inline u32x2 decode4(uint32_t codes, float scale) {
  return (u32x2){Fp8<Tag>::template decode<false>(codes, scale), Fp8<Tag>::template decode<true>(codes, scale)};
}
// Eight codes (two dwords): an MFMA operand.
template <typename Tag>
__device__ inline u32x4 decode8(uint32_t low, uint32_t high, float scale) {
  const u32x2 a = decode4<Tag>(low, scale), b = decode4<Tag>(high, scale);
  return (u32x4){a[0], a[1], b[0], b[1]};
}
template <typename Tag>
__device__ inline uint32_t encode4(uint32_t a, uint32_t b, float scale) {
  shortx2 x = (shortx2){0, 0};
  x = Fp8<Tag>::template encode<false>(x, a, scale);
  x = Fp8<Tag>::template encode<true>(x, b, scale);
  return __builtin_bit_cast(uint32_t, x);
}
// Does one of a dword's four codes stand for NaN?
__device__ inline bool has_nan(uint32_t codes) {
  return (((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
}

__device__ inline uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int s = 1; s < 64; s *= 2) {
    const uint32_t o = __shfl_xor(x, s, 64);
    x = x > o ? x : o;
  }
  return __builtin_amdgcn_readfirstlane(x);
}

// The page of a sequence's column, or -1. `column` lies inside the table.
__device__ inline int page_at(const Kv8Pages& c, int b, int64_t column) {
  const int page = c.table[(int64_t)b * c.columns + column];
  return (uint32_t)page < (uint32_t)c.pages ? page : -1;
}

// Append: a wave takes a block, 16 channels of a row to a lane and step: the tokens that the block holds already, the
// new rows, zeros behind them. The largest finite magnitude of all gives the scale (integer compares: any host that
// follows the definition gets the same bytes), and the block is written whole, so it holds nothing of rows that were
// drafted in vain or of what the page held before, and its scale is that of its tokens. (Tokens that stay are rounded again
// where the scale grows.) Bound by memory: 4 prompts of 2-4k tokens,
// 8 heads, D = 128, values returned (149 MB), 24.5 us, 6.1 TB/s, some of it in the caches. A step of 32 single tokens
// 6 us: a chain of four dependent loads (start, page, the block's scale and codes, all but the last two in turn).
template <typename Tag, int D>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8AppendParams p) {
  typedef Fp8<Tag> F;
  constexpr int UPR = D / 16, PER = 32 * UPR / 64;
  const int lane = threadIdx.x & 63;
  int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (id >= (int64_t)p.B * p.blocks * p.Hkv) return;
  const bool is_v = blockIdx.y != 0;
  const int h = (int)(id % p.Hkv);  // consecutive rows of a projection output [B, S, H, D] are its heads
  id /= p.Hkv;
  const int blk = (int)(id % p.blocks), b = (int)(id / p.blocks);
  const int64_t start = p.start[b];
  int n = p.count != nullptr ? p.count[b] : p.rows;
  n = n < 0 ? 0 : (n > p.rows ? p.rows : n);
  const int64_t at = ((start >> 5) + blk) * 32;  // the block's first token
  if (at >= start + p.rows) return;
  const int64_t low = start > 0 ? start : 0;
  const int64_t high = start + n < p.capacity ? start + n : p.capacity;
  // rows [r0, r1) of the block are new
  const int r0 = (int)(low - at < 0 ? 0 : (low - at > 32 ? 32 : low - at));
  const int r1 = (int)(high - at < 0 ? 0 : (high - at > 32 ? 32 : high - at));
  const Kv8Pages& c = p.cache;
  int page = -1;
  if (r1 > r0) {
    page = page_at(c, b, at >> (5 + c.blocks_log2));
    if (page >= 0 && c.refs[page] != 1) page = -1;
  }
  uint16_t* out = is_v ? p.v_values : p.k_values;
  if (page < 0 && out == nullptr) return;
  const int64_t* st = is_v ? p.sv : p.sk;
  const uint16_t* src = (is_v ? p.v : p.k) + b * st[0] + h * st[1];
  const int sub = (int)(at >> 5) & ((1 << c.blocks_log2) - 1);
  uint8_t* base = c.data + page * c.page_stride;
  uint8_t* codes = base + (((int64_t)(2 * h + is_v) << c.blocks_log2) + sub) * (32 * D);
  uint8_t* scale_byte = base + c.scales_at + 2 * (((int64_t)h << c.blocks_log2) + sub) + is_v;
  u32x4 x[PER][2];
  uint32_t e = 0;
  if (page >= 0) {
    const float old = block_scale<Tag>(*scale_byte);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = lane + 64 * i, row = u / UPR, part = u % UPR;
      x[i][0] = x[i][1] = (u32x4){0, 0, 0, 0};
      if (row >= r0 && row < r1) {
        const uint16_t* from = src + (at + row - start) * st[2] + part * 16;
        x[i][0] = reinterpret_cast<const u32x4*>(from)[0];
        x[i][1] = reinterpret_cast<const u32x4*>(from)[1];
      } else if (row < r0) {
        const u32x4 held = *reinterpret_cast<const u32x4*>(codes + row * D + part * 16);
        x[i][0] = decode8<Tag>(held[0], held[1], old);
        x[i][1] = decode8<Tag>(held[2], held[3], old);
      }
    }
    // the largest magnitude, two channels at a time; magnitudes of a type compare as whole numbers
    ushortx2 both = (ushortx2){0, 0};
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        both = __builtin_elementwise_max(both, __builtin_bit_cast(ushortx2, x[i][j / 4][j % 4] & 0x7fff7fffu));
    uint32_t top = wave_max(both[0] > both[1] ? both[0] : both[1]);
    bool rare = top > F::kMaxBits;
    if (rare) {
      top = 0;  // of the finite ones; the others, and values past the largest code's, are looked for below
#pragma unroll
      for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const uint32_t a = (x[i][j / 8][j % 8 / 2] >> (16 * (j & 1))) & 0x7fffu;
          top = a < F::kInfBits && a > top ? a : top;
        }
      top = wave_max(top);
    }
    const int power = (int)((__float_as_uint(DT<Tag>::to_float((uint16_t)top)) + 0x1fffffu) >> 23) - 8;
    e = power < (int)F::kFloor ? F::kFloor : (power > (int)F::kCeil ? F::kCeil : (uint32_t)power);
    const float scale = scale_of(e);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      u32x4 nan = (u32x4){0, 0, 0, 0};
      if (rare) {  // NaN for what is not finite; values past the largest code's become that
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int sh = 16 * (j & 1);
          const uint32_t word = x[i][j / 8][j % 8 / 2], a = (word >> sh) & 0x7fffu;
          uint32_t to = a > F::kMaxBits ? (a >= F::kInfBits ? 0u : F::kMaxBits) : a;
          if (a < F::kInfBits) to |= (word >> sh) & 0x8000u;
          if (a >= F::kInfBits) nan[j / 4] |= 0x7fu << (8 * (j % 4));
          x[i][j / 8][j % 8 / 2] = (word & ~(0xffffu << sh)) | (to << sh);
        }
      }
      const int u = lane + 64 * i;
      u32x4 held;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        held[j] = encode4<Tag>(x[i][j / 2][2 * (j & 1)], x[i][j / 2][2 * (j & 1) + 1], scale) | nan[j];
      *reinterpret_cast<u32x4*>(codes + (int64_t)u * 16) = held;
      if (out != nullptr) {
        x[i][0] = decode8<Tag>(held[0], held[1], scale);
        x[i][1] = decode8<Tag>(held[2], held[3], scale);
      }
    }
    if (lane == 0) *scale_byte = (uint8_t)e;
  }
  if (out == nullptr) return;
  const int64_t* so = is_v ? p.svv : p.skv;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int u = lane + 64 * i, row = u / UPR, part = u % UPR;
    const int64_t t = at + row - start;
    if (t < 0 || t >= p.rows) continue;
    const bool written = page >= 0 && row >= r0 && row < r1;
    u32x4* to = reinterpret_cast<u32x4*>(out + b * so[0] + h * so[1] + t * so[2] + part * 16);
    to[0] = written ? x[i][0] : (u32x4){0, 0, 0, 0};
    to[1] = written ? x[i][1] : (u32x4){0, 0, 0, 0};
  }
}

// Running softmax of the prompt chunks. A row's weights are 2^(x c - R + bias), R a whole number: the row's largest score,
// in log2 units, when it was last moved. It is moved when the present one is over kLag further, so that the sums are
// rescaled a few times in all and not at every new maximum, by exact powers of two. fp16: weights up to 2^(8 + 7.5) fit,
// and those down to 2^-22 keep all their bits.
constexpr float kLag = 7.f;
template <typename Tag>
__device__ constexpr float lag_bias();
template <>
__device__ constexpr float lag_bias<f16_t>() { return 8.f; }
template <>
__device__ constexpr float lag_bias<bf16_t>() { return 0.f; }
// Beyond this R, x c and R cancel to what their rounding leaves: the difference of the scores is taken first, from the
// score that gave R, which is its product with c as it stands (rounded to a whole number it would be another's).
constexpr float kLargeR = 0x1p20f;
// bias - R of a row whose reference score is m.
template <typename Tag>
__device__ inline float offset_of(float m, float c) {
  const float whole = lag_bias<Tag>() - __builtin_rintf(m * c);
  return fabsf(whole) <= kLargeR ? whole : lag_bias<Tag>() - m * c;
}
// The reference itself: R, or the score that gave it.
struct Reference {
  float at;
  bool score;
  template <typename Tag>
  __device__ static inline Reference of(float m, float off) {
    const bool whole = fabsf(off) <= kLargeR;
    return {whole ? lag_bias<Tag>() - off : m, !whole};
  }
  // Less another one, in log2 units, rounded once: scores are subtracted before they are multiplied, and no product is
  // rounded before it meets an R (to a sixteenth at 2^20: a weight would be off by 4%).
  __device__ inline float less(const Reference& o, float c) const {
    if (score == o.score) return score ? (at - o.at) * c : at - o.at;
    return score ? fmaf(at, c, -o.at) : -fmaf(o.at, c, -at);
  }
};

// n / d for 0 <= n < 2^31 (the host's numbers in fa_kernels.h): with `shift` = ceil(log2 d), 2^32 + multiplier is
// 2^(32 + shift) / d rounded up. Every workgroup runs through its set-up once, from a cold instruction cache: there a
// division by its 35 instructions is 140 bytes of code to fetch, and there were a dozen.
__device__ inline int divide(int n, const Divisor& d) { return (int)((__umulhi(d.multiplier, (uint32_t)n) + (uint32_t)n) >> d.shift); }

// a / b of whole numbers below 2^53, b > 0.
__device__ inline int64_t divide(int64_t a, int64_t b) {
  int64_t q = (int64_t)((double)a / (double)b);
  if (q * b > a) --q;
  if ((q + 1) * b <= a) ++q;
  return q;
}

// The rows that a group of query rows sees. Query rows are (position, head of the group): row r is head r % group at
// position r / group, and a workgroup's rows share its kv head's cache.
struct Rows {
  int rows, live;  // rows of the kv head, and those before count
  int keys;        // of the sequence
  Divisor by_group;
  int64_t start;
  bool causal;
  __device__ inline Rows(const Kv8AttendParams& p, int b) {
    const int n = p.count != nullptr ? p.count[b] : p.M;
    rows = p.M * p.group;
    live = (n < 0 ? 0 : (n > p.M ? p.M : n)) * p.group;
    keys = visible_keys(p.start, p.count, b, p.M, p.capacity);
    by_group = p.by_group;
    start = p.start[b];
    causal = p.causal != 0;
  }
  // keys that row r sees, if it is live
  __device__ inline int sees(int r) const {
    const int64_t e = causal ? start + divide(r, by_group) + 1 : keys;
    return (int)(e < 0 ? 0 : (e > keys ? keys : e));
  }
  // most keys that one of the live rows in [r, r + n) sees, and the fewest (0 if one of them is not live)
  __device__ inline int most(int r, int n) const { return r >= live ? 0 : sees(r + n <= live ? r + n - 1 : live - 1); }
  __device__ inline int least(int r, int n) const { return r + n <= live ? sees(r) : 0; }
  // fewest that a live row sees
  __device__ inline int live_least(int r) const { return r < live ? sees(r) : 0x7fffffff; }
};

// Where a sequence's blocks of one kv head lie, 64 at a time, one to a lane, and their scales. They are read a lane at a
// time, ready to be used: in the loops over tiles they cost neither a load nor arithmetic.
template <typename Tag, int D>
struct Blocks {
  const int* table;
  const uint8_t* data;        // the head's keys in page 0
  const uint8_t* scales;      // and its scale bytes
  int64_t page_stride, half;  // bytes of a page; of a head's keys in one
  int blocks_log2, pages;
  // of the lane's block: bytes from `data` to its keys, in two halves, and its scales. Without a page: page 0, and the
  // keys' scale is negative.
  int at[2];
  float ks, vs;

  __device__ inline Blocks(const Kv8Pages& c, int b, int hk) {
    half = (int64_t)(32 * D) << c.blocks_log2;
    table = c.table + (int64_t)b * c.columns;
    data = c.data + 2 * hk * half;
    scales = c.data + c.scales_at + 2 * ((int64_t)hk << c.blocks_log2);
    page_stride = c.page_stride;
    blocks_log2 = c.blocks_log2;
    pages = c.pages;
    at[0] = at[1] = 0;
    ks = vs = -1.f;
  }
  // The lane's block becomes `mine` (none at or behind `end`). Where it lies is waited for here, its scales where they
  // are first used.
  __device__ inline void look_up(int mine, int end) {
    int page = -1;
    if (mine < end) page = table[mine >> blocks_log2];
    asm volatile("" : "+v"(page));
    const bool there = (uint32_t)page < (uint32_t)pages;
    const int sub = mine & ((1 << blocks_log2) - 1);
    const int64_t base = there ? page * page_stride : 0, place = base + sub * (32 * D);
    at[0] = (int)place;
    at[1] = (int)(place >> 32);
    const uint32_t e = *reinterpret_cast<const uint16_t*>(scales + base + 2 * sub);
    ks = there ? block_scale<Tag>(e & 255u) : -1.f;
    vs = block_scale<Tag>(e >> 8);
  }
  __device__ inline void wait() { asm volatile("" : "+v"(ks), "+v"(vs)); }
  __device__ inline int64_t keys_at(int lane) const {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(at[0], lane) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readlane(at[1], lane) << 32);
  }
  __device__ inline float key_scale(int lane) const { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ks), lane)); }
  __device__ inline float value_scale(int lane) const { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs), lane)); }
};

template <int N, int J = 0, typename Fn>
__device__ inline void for_each(Fn& f) {
  if constexpr (J < N) {
    f(std::integral_constant<int, J>{});
    for_each<N, J + 1>(f);
  }
}

// Attention over the cache, up to 32 query rows to a kv head. A wave holds 16 R query rows (columns of every product)
// and walks 32-key tiles, which are blocks:
//   S^T = K Q^T     A = K rows: lane (key, 16 of each 64 channels) reads its channels and converts them in place
//   O^T += V^T P^T  A = V^T: lane (channels, 8 keys) reads the keys' codes of its D / 16 channels, converts, and
//                   regroups them by channel with byte permutes; P^T is S^T's accumulator as it stands
// so nothing passes through LDS but the waves' sums at the end. P is rounded to the type once, on its way to the second
// product, as the prompt chunks' is: weights in two 16-bit halves would double that product and P's registers. Sums and
// lse take the unrounded weights. Results are off from 64 bits by 1.9e-3 (bf16) and 2.4e-4 (fp16) of their norm, chunks' by
// 2.3e-3 and 2.9e-4, where fp32 weights and the result's rounding alone leave 1.6e-3 and 2.1e-4.
// A lane keeps the table entries of its wave's next 64 tiles, so that a page number costs no load in the loop; a tile
// without a page is one that no row sees.
// The four waves hold the same rows and take turns at the tiles. A wave has one tile's registers: the next tile's keys are
// asked for when the scores stand, its values when the second product does, so that half a tile or more is in flight.
// Bound by memory where there is enough of it: 8 sequences of 16-32k keys, 8 kv heads, D = 128 (419 MB), 78 us, 5.4 TB/s.
// One sequence of 8k keys: 7.6 us, launch and dependent loads; 4 of 41-65k keys, 2 kv heads, D = 64 (55 MB) 17 us and 3 of
// 12k, 4 heads, D = 256 (76 MB) 18.6: few tiles to a wave, behind the same start.
template <typename Tag, int D, int R>
struct Kv8Attend {
  static constexpr int WAVES = 4;
  static constexpr int KS = D / 32;   // k = 32 steps over D
  static constexpr int CPL = D / 16;  // channels of V per lane
  static constexpr int KW = D / 16;   // dwords of K codes per lane and key
  static constexpr int VW = CPL / 4;  // dwords of V codes per lane and key
  typedef DT<Tag> E;
  typedef Fp8<Tag> F;

  // One lane's share of a block, as stored.
  typedef uint32_t Keys[2][KW];
  typedef uint32_t Values[8][VW];

  __device__ static inline void load_keys(Keys& k, const uint8_t* from, int lane) {
    from += (uint32_t)((lane & 15) * D + 16 * (lane >> 4));
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(from + 16 * i * D + 64 * j);
#pragma unroll
        for (int w = 0; w < 4; ++w) k[i][4 * j + w] = x[w];
      }
  }
  // Keys of a lane's k-slots in the second product: slot i is key 4 g + (i & 3) + 16 (i >> 2).
  __device__ static inline void load_values(Values& v, const uint8_t* from, int lane) {
    from += (uint32_t)(4 * (lane >> 4) * D + (lane & 15) * CPL);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint8_t* at = from + ((i & 3) + 16 * (i >> 2)) * D;
      if constexpr (VW == 1) {
        v[i][0] = *reinterpret_cast<const uint32_t*>(at);
      } else {
        typedef uint32_t words_t __attribute__((ext_vector_type(VW)));
        const words_t x = *reinterpret_cast<const words_t*>(at);
#pragma unroll
        for (int w = 0; w < VW; ++w) v[i][w] = x[w];
      }
    }
  }

  struct State {
    floatx4 o[CPL][R];
    float m[R], l[R];
  };

  // The n-th key's values times P, if it is marked in `bad`: a product of its own, whose result only the rows that see
  // the key take.
  __device__ static inline void add_alone(State& s, const Values& v, float scale, const u32x4 (&pb)[R], uint32_t bad, int n,
                                          int key0, const int (&see)[R], int lane) {
    const int slot = (n & 3) + 4 * (n >> 4);
    const bool mine = lane >> 4 == ((n >> 2) & 3) && (bad >> slot & 1u) != 0;
    if (!__any(mine)) return;
    uint32_t code[VW] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i == slot) {
#pragma unroll
        for (int w = 0; w < VW; ++w) code[w] = v[i][w];
      }
    auto pair = [&](auto jc) {
      constexpr int j = decltype(jc)::value;
      const uint32_t x = mine ? F::template decode<(j & 1) != 0>(code[j / 2], scale) : 0u;
      u32x4 even, odd;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        even[i] = i == slot / 2 ? (x & 0xffffu) << (16 * (slot & 1)) : 0u;
        odd[i] = i == slot / 2 ? (x >> 16) << (16 * (slot & 1)) : 0u;
      }
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        const floatx4 zero = (floatx4){0.f, 0.f, 0.f, 0.f};
        const floatx4 a = E::mfma16(even, pb[rt], zero), b = E::mfma16(odd, pb[rt], zero);
        if (key0 + n < see[rt]) {
          s.o[2 * j][rt] += a;
          s.o[2 * j + 1][rt] += b;
        }
      }
    };
    for_each<CPL / 2>(pair);
  }

  // One tile: keys [key0, key0 + 32), of which row rt sees those below see[rt] (a lane's own row). ks, vs: its scales.
  // there: they have a page (`keys` is 0 otherwise). `edge`: a row does not see all of them; `unseen`: a live row does not see all of the sequence's keys among them.
  // next_keys() and next_values() ask for the next tile's codes as soon as this one's have been used. (One body with
  // branches for the edge: with a body of its own for whole tiles the registers of both are held, and 60 spilled.)
  template <typename NextKeys, typename NextValues>
  __device__ static inline void step(State& s, const u32x4 (&qf)[R][KS], const Keys& kc, Values& vc, float ks, float vs,
                                     int key0, const int (&see)[R], int keys, bool there, bool edge, bool unseen, float c, int lane,
                                     NextKeys&& next_keys, NextValues&& next_values) {
    const int g = lane >> 4;
    floatx4 x[2][R];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int rt = 0; rt < R; ++rt) x[i][rt] = (floatx4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const u32x4 a = decode8<Tag>(kc[i][2 * k], kc[i][2 * k + 1], ks);
#pragma unroll
        for (int rt = 0; rt < R; ++rt) x[i][rt] = E::mfma16(a, qf[rt][k], x[i][rt]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    next_keys();
    __builtin_amdgcn_sched_barrier(0);
    u32x4 pb[R];
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      if (edge) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key0 + 16 * i + 4 * g + r >= see[rt] || !there) x[i][rt][r] = FA_NEG_INF;
      }
      // a NaN score makes the row NaN: through P, whether or not the maximum moves
      const float top = larger(larger(larger(x[0][rt][0], x[0][rt][1]), larger(x[0][rt][2], x[0][rt][3])),
                               larger(larger(x[1][rt][0], x[1][rt][1]), larger(x[1][rt][2], x[1][rt][3])));
      const float m_new = larger(s.m[rt], row_max(top));
      if (__any(m_new > s.m[rt])) {
        const float base = m_new == FA_NEG_INF ? 0.f : m_new;
        const float f = fast_exp2((s.m[rt] - base) * c);
        s.l[rt] *= f;
#pragma unroll
        for (int d = 0; d < CPL; ++d) s.o[d][rt] *= f;
        s.m[rt] = m_new;
      }
      const float base = s.m[rt] == FA_NEG_INF ? 0.f : s.m[rt];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[i][rt][r] = fast_exp2(fmaf(x[i][rt][r] - base, c, weight_bias<Tag>()));
          s.l[rt] += x[i][rt][r];
        }
      pb[rt] = (u32x4){E::pack2(x[0][rt][0], x[0][rt][1]), E::pack2(x[0][rt][2], x[0][rt][3]),
                       E::pack2(x[1][rt][0], x[1][rt][1]), E::pack2(x[1][rt][2], x[1][rt][3])};
    }
    if (edge) {
      // Rows behind the last key may hold anything, NaN too: they read as zeros. A NaN would be 0 x NaN to the rows
      // that do not see its key: keys that have one (rare) leave the tile's product and are added one by one.
      uint32_t bad = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool behind = key0 + 4 * g + (i & 3) + 16 * (i >> 2) >= keys;
        bool nan = false;
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          if (behind) vc[i][w] = 0;
          nan |= has_nan(vc[i][w]);
        }
        bad |= (nan ? 1u : 0u) << i;
      }
      if (!unseen) bad = 0;
      if (__builtin_expect(__any(bad != 0), 0)) {
#pragma unroll 1
        for (int n = 0; n < 32; ++n) add_alone(s, vc, vs, pb, bad, n, key0, see, lane);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (bad >> i & 1u) {
#pragma unroll
            for (int w = 0; w < VW; ++w) vc[i][w] = 0;
          }
      }
    }
    // channels 2 j and 2 j + 1 of the lane's CPL
    auto pair = [&](auto jc) {
      constexpr int j = decltype(jc)::value;
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = F::template decode<(j & 1) != 0>(vc[i][j / 2], vs);
      u32x4 even, odd;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        even[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100u);
        odd[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302u);
      }
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        s.o[2 * j][rt] = E::mfma16(even, pb[rt], s.o[2 * j][rt]);
        s.o[2 * j + 1][rt] = E::mfma16(odd, pb[rt], s.o[2 * j + 1][rt]);
      }
    };
    for_each<CPL / 2>(pair);
    __builtin_amdgcn_sched_barrier(0);
    next_values();
  }

  // N channels N at .. of row r, whose maximum and sum are m and l. A row that saw no key (l = 0) is zeros, whatever its
  // products with values that are no numbers left in o.
  template <int N>
  __device__ static inline void store_row(const Kv8AttendParams& p, int b, int hk, int slot, int r, const float (&o)[N],
                                          float m, float l, int at) {
    const int i = divide(r, p.by_group), h = hk * p.group + r - i * p.group;
    if (p.splits > 1) {
      const int64_t w = ((int64_t)slot * p.H + h) * p.M + i;
      float* dst = p.ws_o + w * D + at * N;
#pragma unroll
      for (int j = 0; j < N; j += 4)
        *reinterpret_cast<floatx4*>(dst + j) =
            l == 0.f ? (floatx4){0.f, 0.f, 0.f, 0.f} : (floatx4){o[j], o[j + 1], o[j + 2], o[j + 3]};
      if (at == 0) {
        p.ws_ml[2 * w] = m;
        p.ws_ml[2 * w + 1] = l;
      }
    } else {
      const float inv = 1.f / l;
      uint16_t* dst = p.o + b * p.so[0] + h * p.so[1] + i * p.so[2] + at * N;
#pragma unroll
      for (int j = 0; j < N; j += 4)
        *reinterpret_cast<u32x2*>(dst + j) = l == 0.f ? (u32x2){0u, 0u}
                                                      : (u32x2){E::pack2(o[j] * inv, o[j + 1] * inv),
                                                                E::pack2(o[j + 2] * inv, o[j + 3] * inv)};
      if (at == 0 && p.lse != nullptr)
        p.lse[b * p.sl[0] + h * p.sl[1] + i * p.sl[2]] =
            l == 0.f ? FA_NEG_INF : (m * p.c + __builtin_amdgcn_logf(l) - weight_bias<Tag>()) * 0.6931471805599453f;
    }
  }

  __device__ static void run(const Kv8AttendParams& p, float* smem) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    // row blocks innermost: those of one split share its tiles in L2
    const int rest = divide(id, p.by_blocks), rb = id - rest * p.row_blocks;
    const int hk = divide(rest, p.by_slots), slot = rest - hk * p.slots;
    const Split part = find_split(p, slot, 0);
    const int b = __builtin_amdgcn_readfirstlane(part.b);
    if (b < 0) return;
    const Rows q_rows(p, b);
    const int row0 = rb * 16 * R, keys = q_rows.keys;

    int see[R];  // keys that the lane's row sees
    u32x4 qf[R][KS];
    State s;
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      const int r = row0 + 16 * rt + c16;
      const bool live = r < q_rows.live;
      see[rt] = live ? q_rows.sees(r) : 0;
      const int pos = live ? divide(r, p.by_group) : 0, member = live ? r - pos * p.group : 0;
      const uint16_t* q = p.q + b * p.sq[0] + (int64_t)(hk * p.group + member) * p.sq[1] + pos * p.sq[2] + g * 16;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qf[rt][k] = (u32x4){0, 0, 0, 0};
        if (live) qf[rt][k] = *reinterpret_cast<const u32x4*>(q + 64 * (k / 2) + 8 * (k & 1));
      }
      s.m[rt] = FA_NEG_INF;
      s.l[rt] = 0.f;
#pragma unroll
      for (int d = 0; d < CPL; ++d) s.o[d][rt] = (floatx4){0.f, 0.f, 0.f, 0.f};
    }
    const int least = __builtin_amdgcn_readfirstlane(q_rows.least(row0, 16 * R));
    const int live_least = __builtin_amdgcn_readfirstlane(q_rows.live_least(row0));
    const int tiles = (__builtin_amdgcn_readfirstlane(q_rows.most(row0, 16 * R)) + 31) / 32;
    const int per = __builtin_amdgcn_readfirstlane(part.per);
    const int64_t first = (int64_t)__builtin_amdgcn_readfirstlane(part.index) * per;
    const int t1 = __builtin_amdgcn_readfirstlane((int)(first + per < tiles ? first + per : tiles));
    const int t0 = __builtin_amdgcn_readfirstlane(first < t1 ? (int)first + wave : t1);
    Blocks<Tag, D> blocks(p.cache, b, hk);  // of the wave's next 64 tiles
    // Codes are asked for without a condition, so that a wait for one load need not be a wait for all behind it: where
    // there is no next tile the last one is read again (from L2), where it has no page page 0 is.
    if (t0 < t1) {
      blocks.look_up(t0 + lane * WAVES, t1);
      int used = 0;  // of the 64
      Keys kc;
      Values vc;
      int64_t at = blocks.keys_at(0);  // of the next tile's keys
      auto next_keys = [&]() { load_keys(kc, blocks.data + at, lane); };
      auto next_values = [&]() { load_values(vc, blocks.data + blocks.half + at, lane); };
      next_keys();
      next_values();
      blocks.wait();
      for (int t = t0; t < t1; t += WAVES) {
        const float ks = blocks.key_scale(used), vs = blocks.value_scale(used);
        const bool there = ks >= 0.f;
        if (t + WAVES < t1) {
          if (++used == 64) {
            blocks.look_up(t + WAVES + lane * WAVES, t1);
            blocks.wait();
            used = 0;
          }
          at = blocks.keys_at(used);
        }
        step(s, qf, kc, vc, ks, vs, t * 32, see, there ? keys : 0, there, t * 32 + 32 > least || !there,
             (t * 32 + 32 < keys ? t * 32 + 32 : keys) > live_least, p.c, lane, next_keys, next_values);
      }
    }
    // the waves' sums meet in LDS; wave w finishes rows 4 w .. 4 w + 3 of each 16, 16 lanes to a row
    constexpr int ROW = D + 4;
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      const float l = xquad_sum(s.l[rt]);
      float* dst = smem + (wave * 16 + c16) * ROW;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int d = 0; d < CPL; d += 4)
          *reinterpret_cast<floatx4*>(dst + (4 * g + r) * CPL + d) =
              (floatx4){s.o[d][rt][r], s.o[d + 1][rt][r], s.o[d + 2][rt][r], s.o[d + 3][rt][r]};
      if (g == 0) {
        dst[D] = s.m[rt];
        dst[D + 1] = l;
      }
      __syncthreads();
      const int row = 4 * wave + g;
      float m = FA_NEG_INF;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) m = fmaxf(m, smem[(w * 16 + row) * ROW + D]);
      float sum = 0.f, o[CPL];
#pragma unroll
      for (int j = 0; j < CPL; ++j) o[j] = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float* src = smem + (w * 16 + row) * ROW;
        const float f = m == FA_NEG_INF ? 1.f : fast_exp2((src[D] - m) * p.c);
        sum += f * src[D + 1];
#pragma unroll
        for (int j = 0; j < CPL; ++j) o[j] = fmaf(f, src[c16 * CPL + j], o[j]);
      }
      const int r = row0 + 16 * rt + row;
      if (r < q_rows.rows) store_row<CPL>(p, b, hk, slot, r, o, m, sum, c16);
      __syncthreads();
    }
  }
};

// Waves per SIMD: what the registers of a tile, Q and O allow without spilling.
template <int D, int R>
constexpr int attend8_waves() {
  return D == 64 ? (R == 1 ? 5 : 3) : (D == 128 && R == 1 ? 4 : 2);
}
template <typename Tag, int D, int R>
__global__ __launch_bounds__(256, (attend8_waves<D, R>())) void kv8_attend_kernel(Kv8AttendParams p) {
  __shared__ __align__(16) float smem[4 * 16 * (D + 4)];
  Kv8Attend<Tag, D, R>::run(p, smem);
}
// The kernel of 32 rows. At D = 256 a tile, Q and O of 32 rows take more registers than a wave has (144 spilled): there
// workgroups of 16 rows lie next to each other and the second reads the cache from L2. 24 rows against 16k keys, one
// sequence: 23.3 us against 22.8, 8 sequences 63 against 61; prompts' kernel 48 and 75.
template <typename Tag, int D>
constexpr const void* attend_two_tiles() {
  if constexpr (D == 256) return nullptr;
  else return (const void*)&kv8_attend_kernel<Tag, D, 2>;
}

// Chunks of a prompt: more than 32 query rows to a kv head. The workgroup's four waves, of 32 rows each, share the
// conversion: a tile's codes are loaded a tile ahead, 16 channels of a row to a thread and step, converted once into
// 16-bit rows in LDS (two stages, one barrier a tile), and both products read their fragments there, V's by the
// transposing read. S^T = K Q^T and O^T = V^T P^T as above. The chip's workgroups take equal shares of all blocks' tiles,
// or whole blocks where there are at least two to a place, the longest first (both sides measured at kv8_attend_splits).
// Products of 1024 rows against 32k keys, 32/8 heads, bf16, D = 128 run at 970 to 1000 TFLOP/s by card, of a first 2048 rows
// at 770, fp16 D = 64 at 690 and D = 256 at 755. Bound by two waves to a SIMD (registers, LDS): matrix unit, vector unit and
// LDS are busy about half of the time each, and overlap as far as two waves let them. Eight waves in two groups that take
// turns at products and softmax were 5 to 25% slower than four (without fragments ahead), their barriers cost more than the
// overlap gave.
// Sums of the rounded weights by the matrix unit gave 1 to 5% and an lse of 16-bit weights: the sums stay in the vector unit.

// Fewest key tiles to a workgroup's share: below, the parts' extra pass costs more than it gives.
constexpr int kMinShare = 4;

template <typename Tag, int D>
struct Kv8Chunk {
  using L = LdsRows<D>;
  typedef DT<Tag> E;
  typedef Fp8<Tag> F;
  static constexpr int WAVES = 4, QT = D == 256 ? 1 : 2;  // 16-row tiles of queries per wave
  static constexpr int T = D == 256 ? 32 : 64;  // keys of a tile
  static constexpr int NB = T / 32;             // its blocks
  static constexpr int KT = T / 16, KS = D / 32, DT16 = D / 16, UPR = D / 16;
  static constexpr int BLOCK = WAVES * QT * 16;
  static constexpr int TILEB = T * L::ROWB, STAGEB = 2 * TILEB;
  static constexpr int SMEM = 2 * STAGEB;
  // Fragments in flight, as the registers allow: at D = 128 (255 of them in bf16, all 256 in fp16) 244 us with 8 for 2 x 28
  // heads of 509 rows, 252 with 4; at D = 256 709 us with 8 for 2 x 16 heads of 1024, 701 with 4; at D = 64 4 spills ten
  // registers in bf16, 3 spills four (five in fp16).
  static constexpr int kAhead = D == 64 ? 3 : (D == 128 ? 8 : 4);
  static constexpr int PER = T * UPR / 256;  // 16-channel units of K, and of V, per thread
  static_assert(PER * 256 == T * UPR, "units");

  struct Codes {
    u32x4 k[PER], v[PER];
    float ks[NB], vs[NB];  // scales of the tile's blocks; ks < 0: it has no page
  };

  // block of the tile that a wave's i-th unit lies in
  __device__ static inline int block_of(int i, int wave) { return D == 128 ? i : (D == 64 ? wave >> 1 : 0); }

  // The work of all row blocks, head after head, is a line of key tiles: block rb of sequence b has as many as its rows
  // see. (One at least: blocks without live rows have zeros to write.) A pair is b * row_blocks + rb.
  __device__ static inline int tiles_of(const Kv8AttendParams& p, int pair) {
    const int b = divide(pair, p.by_blocks);
    const Rows rows(p, b);
    const int n = (rows.most((pair - b * p.row_blocks) * BLOCK, BLOCK) + T - 1) / T;
    return n > 0 ? n : 1;
  }
  // Tiles of a head's pairs up to the one that holds tile `at` (and that pair), or of all. 64 pairs at a time, one to a
  // lane; every wave works it out for itself.
  struct Place {
    int pair;
    int64_t before;
  };
  typedef uint32_t Tiles;
  static_assert((uint64_t)(kMaxCapacity / T) * 64 <= std::numeric_limits<Tiles>::max(), "64 row blocks of the longest sequence");
  __device__ static inline Place find(const Kv8AttendParams& p, int64_t at) {
    const int lane = threadIdx.x & 63, pairs = p.B * p.row_blocks;
    int64_t base = 0;
    for (int c = 0; c < pairs; c += 64) {
      const Tiles n = c + lane < pairs ? (Tiles)tiles_of(p, c + lane) : 0;
      Tiles end = n;
#pragma unroll
      for (int k = 1; k < 64; k *= 2) {
        const Tiles o = __shfl_up(end, k, 64);
        if (lane >= k) end += o;
      }
      const uint64_t hit = __ballot(at < base + end);
      if (hit != 0) {
        const int who = __builtin_ctzll(hit);
        return {c + who, base + (Tiles)__builtin_amdgcn_readlane((int)(end - n), who)};
      }
      base += (Tiles)__builtin_amdgcn_readlane((int)end, 63);
    }
    return {pairs, base};
  }

  // One workgroup: a row block (splits = 1; the longest first), or an equal share of the line, whose ends may lie inside
  // a block: such parts are left in the workspace, the share's first part (which continues a block) in slot 2 id and its
  // last (which begins one) in slot 2 id + 1.
  // flags: words with a bit for each key of the tile whose values hold a NaN, for three tiles in turn
  __device__ static void run(const Kv8AttendParams& p, char* smem, uint32_t (*flags)[2]) {
    const int pairs = p.B * p.row_blocks;
    const bool shared = p.splits > 1;
    const int id = shared ? xcd_remap(blockIdx.x, gridDim.x) : (int)blockIdx.x;
    if (threadIdx.x < 6) flags[threadIdx.x / 2][threadIdx.x % 2] = 0;
    __syncthreads();
    Turn turn = {0, 0};
    int hk, pair;
    int64_t at = 0, end = 1, begun = 0, share = 1;  // on the line; of the pair's tiles
    if (shared) {
      const int64_t all = find(p, INT64_MAX).before, line = all * p.Hkv;
      share = divide(line + gridDim.x - 1, (int64_t)gridDim.x);
      if (share < kMinShare) share = kMinShare;
      at = id * share;
      end = at + share < line ? at + share : line;
      if (at >= end) return;
      hk = (int)divide(at, all);
      const Place place = find(p, at - hk * all);
      pair = place.pair;
      begun = at - hk * all - place.before;
    } else {
      const int from_last = divide(id, p.by_slots), rest = id - from_last * p.slots;  // slots: heads of all sequences
      hk = rest % p.Hkv;
      pair = rest / p.Hkv * p.row_blocks + p.row_blocks - 1 - from_last;
    }
    hk = __builtin_amdgcn_readfirstlane(hk);
    pair = __builtin_amdgcn_readfirstlane(pair);
    while (at < end) {
      const int n = __builtin_amdgcn_readfirstlane(tiles_of(p, pair));
      const int t0 = __builtin_amdgcn_readfirstlane((int)begun);
      const int t1 = __builtin_amdgcn_readfirstlane((int)(shared && end - at < n - t0 ? t0 + (end - at) : n));
      const int b = __builtin_amdgcn_readfirstlane(divide(pair, p.by_blocks));
      part(p, smem, flags, turn, hk, b, pair - b * p.row_blocks, t0, t1, t0 == 0 && t1 == n ? -1 : 2 * id + (t0 == 0));
      if (shared && t1 == n && threadIdx.x == 0) {  // who has the block's parts: the first workgroup, and how many
        const int first = (int)divide(at - t0, share);
        p.parts[2 * (hk * (int64_t)pairs + pair)] = first;
        p.parts[2 * (hk * (int64_t)pairs + pair) + 1] = id - first + 1;
      }
      at += t1 - t0;
      begun = 0;
      if (++pair == pairs) {
        pair = 0;
        ++hk;
      }
    }
  }

  struct Turn {  // LDS stage and flags' turn: they go on from part to part
    uint32_t stage;
    int flag;
  };

  // Tiles [t0, t1) of row block rb, for one kv head of one sequence. slot: -1, or where the sums are left.
  __device__ static void part(const Kv8AttendParams& p, char* smem, uint32_t (*flags)[2], Turn& at_turn, int hk, int b, int rb,
                              int t0, int t1, int slot) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    const Rows q_rows(p, b);
    const int row0 = rb * BLOCK + wave * QT * 16, keys = q_rows.keys;
    const int block_see = __builtin_amdgcn_readfirstlane(q_rows.most(rb * BLOCK, BLOCK));
    const int wave_see = __builtin_amdgcn_readfirstlane(q_rows.most(row0, QT * 16));
    const int least = __builtin_amdgcn_readfirstlane(q_rows.least(row0, QT * 16));
    const int block_least = __builtin_amdgcn_readfirstlane(q_rows.live_least(rb * BLOCK));

    int see[QT];
    u32x4 qf[QT][KS];
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      const int r = row0 + 16 * j + c16;
      const bool live = r < q_rows.live;
      see[j] = live ? q_rows.sees(r) : 0;
      const int pos = live ? divide(r, p.by_group) : 0, member = live ? r - pos * p.group : 0;
      const uint16_t* q = p.q + b * p.sq[0] + (int64_t)(hk * p.group + member) * p.sq[1] + pos * p.sq[2] + 8 * g;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qf[j][k] = (u32x4){0, 0, 0, 0};
        if (live) qf[j][k] = *reinterpret_cast<const u32x4*>(q + 32 * k);
      }
    }
    floatx4 o[DT16][QT];
    float m[QT], l[QT], off[QT];  // row's reference score, sum of weights, bias - R
    bool large = false;
    const float lag = fminf(kLag / p.c, 0x1.fffffep127f);  // finite, so that any score moves the first maximum
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      m[j] = FA_NEG_INF;
      l[j] = 0.f;
      off[j] = lag_bias<Tag>();
#pragma unroll
      for (int d = 0; d < DT16; ++d) o[d][j] = (floatx4){0.f, 0.f, 0.f, 0.f};
    }

    const int k_first = t0 * T;
    const int k_end = t1 * T < block_see ? t1 * T : block_see;  // t1 * T <= the capacity rounded up, under 2^31
    int live_least = __builtin_amdgcn_readfirstlane(q_rows.live_least(row0));
    if (live_least < 0x7fffffff && live_least > k_end) live_least = k_end;
    Blocks<Tag, D> blocks(p.cache, b, hk);
    const int end = (k_end + 31) / 32;
    int used = 0;
    if (k_first < k_end) blocks.look_up(k_first / 32 + lane, end);
    // Whole blocks are read, from page 0 where there is no page; what is not to be seen is cleared when it is converted.
    auto fetch = [&](Codes& x, int key0) {
      if (used == 64) {
        blocks.look_up(key0 / 32 + lane, end);
        blocks.wait();
        used = 0;
      }
      const uint8_t* from[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        from[n] = blocks.data + blocks.keys_at(used + n);
        x.ks[n] = blocks.key_scale(used + n);
        x.vs[n] = blocks.value_scale(used + n);
      }
      used += NB;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int n = block_of(i, wave);
        const uint8_t* at = (NB == 2 && n ? from[NB - 1] : from[0]) + (uint32_t)((tid + 256 * i) / UPR % 32 * D + tid % UPR * 16);
        x.k[i] = *reinterpret_cast<const u32x4*>(at);
        x.v[i] = *reinterpret_cast<const u32x4*>(at + blocks.half);
      }
    };
    // `mark`: the tile has keys that one of the workgroup's live rows does not see
    // Keys behind the last one that any row sees may hold anything, NaN too: their values read as zeros.
    auto convert = [&](Codes& x, int key0, uint32_t stage, int turn, bool mark) {
      bool clear = key0 + T > keys;
#pragma unroll
      for (int n = 0; n < NB; ++n) clear = clear || x.ks[n] < 0.f;
      if (clear) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int n = block_of(i, wave);
          const bool gone = (NB == 2 && n ? x.ks[NB - 1] : x.ks[0]) < 0.f;
          if (gone || key0 + (tid + 256 * i) / UPR >= keys) x.v[i] = (u32x4){0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int row = (tid + 256 * i) / UPR, part16 = tid % UPR;
        const int n = block_of(i, wave);
        char* dst = smem + stage + row * L::ROWB;
        const uint32_t c0 = (uint32_t)(((2 * part16) ^ L::swz(row)) << 4), c1 = (uint32_t)(((2 * part16 + 1) ^ L::swz(row)) << 4);
        const float ks = NB == 2 && n ? x.ks[NB - 1] : x.ks[0], vs = NB == 2 && n ? x.vs[NB - 1] : x.vs[0];
        *reinterpret_cast<u32x4*>(dst + c0) = decode8<Tag>(x.k[i][0], x.k[i][1], ks);
        *reinterpret_cast<u32x4*>(dst + c1) = decode8<Tag>(x.k[i][2], x.k[i][3], ks);
        *reinterpret_cast<u32x4*>(dst + TILEB + c0) = decode8<Tag>(x.v[i][0], x.v[i][1], vs);
        *reinterpret_cast<u32x4*>(dst + TILEB + c1) = decode8<Tag>(x.v[i][2], x.v[i][3], vs);
        if (mark && (has_nan(x.v[i][0]) || has_nan(x.v[i][1]) || has_nan(x.v[i][2]) || has_nan(x.v[i][3])))
          atomicOr(&flags[turn][row >> 5], 1u << (row & 31));
      }
    };
    const uint32_t ro = L::row_off(lane), to = L::tr_off(lane);
    auto step = [&](int key0, uint32_t stage, const bool (&there)[NB], int turn, auto edge_tile) {
      constexpr bool EDGE = decltype(edge_tile)::value;
      const uint32_t rowb = ro + stage, colb = to + stage;
      // A NaN would be 0 x NaN to the rows that do not see its key: keys that have one (rare) are left out of the tile's
      // product and added one by one, to the rows that see them.
      uint64_t alone = 0;  // keys of the tile
      if (EDGE && (key0 + T < keys ? key0 + T : keys) > live_least)
        alone = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)flags[turn][0]) |
                (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)flags[turn][1]) << 32;
      // Fragments are asked for kAhead before their products, in this order: left to itself the compiler asks for each right
      // before its two products and waits for it, an LDS latency for every 32 cycles of the matrix unit.
      u32x4 ring[kAhead];
      auto keys_of = [&](int n) { return L::frag(smem, rowb ^ (n % KS << 6), n / KS * 16 * L::ROWB); };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) ring[n] = keys_of(n);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);  // before a neighbour's softmax
      floatx4 x[KT][QT];
#pragma unroll
      for (int n = 0; n < KT * KS; ++n) {
        const int i = n / KS, k = n % KS;
#pragma unroll
        for (int j = 0; j < QT; ++j)
          x[i][j] = E::mfma16(ring[n % kAhead], qf[j][k], k == 0 ? (floatx4){0.f, 0.f, 0.f, 0.f} : x[i][j]);
        if (n + kAhead < KT * KS) ring[n % kAhead] = keys_of(n + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      bool move[QT];
      float tops[QT];
#pragma unroll
      for (int j = 0; j < QT; ++j) {
        float top = FA_NEG_INF;
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (EDGE && (key0 + 16 * i + 4 * g + r >= see[j] || !there[i / 2])) x[i][j][r] = FA_NEG_INF;
            top = larger(top, x[i][j][r]);
          }
        tops[j] = row_max(top);
        // the difference, not the sum m + lag: that one rounds to the spacing of the scores. A NaN score makes the row NaN
        // through P
        move[j] = tops[j] - m[j] > lag;
      }
      if (__any(QT == 2 ? move[0] || move[QT - 1] : move[0])) {
        bool far = false;
#pragma unroll
        for (int j = 0; j < QT; ++j) {
          // each row by itself: what another row of the wave sees does not change its bits
          float to = offset_of<Tag>(tops[j], p.c);
          float back = to - off[j];
          if (__builtin_expect(__any(!(fmaxf(fabsf(to), fabsf(off[j])) <= kLargeR)), 0))
            back = Reference::of<Tag>(m[j], off[j]).less(Reference::of<Tag>(tops[j], to), p.c);
          const float f = m[j] == FA_NEG_INF ? 0.f : (move[j] ? fast_exp2(back) : 1.f);
          to = move[j] ? to : off[j];
          l[j] *= f;
#pragma unroll
          for (int d = 0; d < DT16; ++d) o[d][j] *= f;
          m[j] = move[j] ? tops[j] : m[j];
          off[j] = to;
          far |= !(fabsf(to) <= kLargeR);
        }
        large = __any(far);
      }
      float add[QT];
#pragma unroll
      for (int j = 0; j < QT; ++j) add[j] = off[j];
      if (__builtin_expect(large, 0)) {
#pragma unroll
        for (int j = 0; j < QT; ++j) {
          const bool far = !(fabsf(off[j]) <= kLargeR);
          add[j] = far ? lag_bias<Tag>() : off[j];
#pragma unroll
          for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int n = 0; n < 4; ++n) x[i][j][n] -= far ? m[j] : 0.f;
        }
      }
      constexpr int VALUES = DT16 * KT / 2;
      auto values_of = [&](int n) { return L::tfrag(smem, colb ^ (n / (KT / 2) << 5), TILEB + n % (KT / 2) * 32 * L::ROWB); };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) ring[n] = values_of(n);
      __builtin_amdgcn_sched_barrier(0);
      u32x4 pb[KT / 2][QT];
#pragma unroll
      for (int j = 0; j < QT; ++j)
#pragma unroll
        for (int i = 0; i < KT; ++i) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[i][j][r] = fast_exp2(fmaf(x[i][j][r], p.c, add[j]));
            l[j] += x[i][j][r];
          }
          pb[i / 2][j][2 * (i & 1)] = E::pack2(x[i][j][0], x[i][j][1]);
          pb[i / 2][j][2 * (i & 1) + 1] = E::pack2(x[i][j][2], x[i][j][3]);
        }
      // a lane's keys of an operand that are in `set`: 4 g .. + 3 (dwords 0, 1), then 16 further (dwords 2, 3)
      auto lanes_of = [&](uint32_t set) {
        const uint32_t x = set >> (4 * g);
        u32x4 m;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint32_t two = x >> (16 * (n / 2) + 2 * (n & 1));
          m[n] = (two & 1u ? 0xffffu : 0u) | (two & 2u ? 0xffff0000u : 0u);
        }
        return m;
      };
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int n = 0; n < VALUES; ++n) {
        const int d = n / (KT / 2), i = n % (KT / 2);
        u32x4 v = ring[n % kAhead];
        if (EDGE && alone != 0) v &= ~lanes_of((uint32_t)(alone >> (32 * i)));
#pragma unroll
        for (int j = 0; j < QT; ++j) o[d][j] = E::mfma16(v, pb[i][j], o[d][j]);
        if (n + kAhead < VALUES) ring[n % kAhead] = values_of(n + kAhead);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      if constexpr (EDGE) {
#pragma unroll 1
        for (; alone != 0; alone &= alone - 1) {
          const int key = __builtin_ctzll(alone), i = key / 32;
          const u32x4 one = lanes_of(1u << (key & 31));
          uint32_t cols = colb + (uint32_t)(i * 32 * L::ROWB);
          asm volatile("" : "+v"(cols));  // addresses worked out here, not held through the loops
#pragma unroll
          for (int j = 0; j < QT; ++j) {
            u32x4 w;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const uint32_t low = pb[0][j][n], high = pb[KT / 2 - 1][j][n];
              w[n] = i != 0 ? high : low;
            }
#pragma unroll
            for (int d = 0; d < DT16; ++d) {
              __builtin_amdgcn_sched_barrier(0);  // nor reads ahead
              const u32x4 v = L::tfrag(smem, cols ^ (d << 5), TILEB) & one;
              const floatx4 x = E::mfma16(v, w, (floatx4){0.f, 0.f, 0.f, 0.f});
              if (key0 + key < see[j]) o[d][j] += x;
            }
          }
        }
      }
    };
    Codes next;
    if (k_first < k_end) fetch(next, k_first);
    uint32_t stage = at_turn.stage;
    int turn = at_turn.flag;
    // Tiles that every row of the wave sees whole, up to a missing page; then the rest, on the diagonal, at the end or
    // with pages missing: every wave makes the same number of passes in all, for the barriers.
    auto pass = [&](int key0, auto edge_tile) {
      bool there[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) there[n] = next.ks[n] >= 0.f;
      convert(next, key0, stage, turn, key0 + T > block_least);
      if (key0 + T < k_end) fetch(next, key0 + T);
      const int after = turn == 2 ? 0 : turn + 1;
      if (tid < 2) flags[after][tid] = 0;  // last read two barriers ago, written again after the next
      wait_vm_lds_barrier<63>();  // LDS writes only: the codes just asked for stay in flight
      if (key0 < wave_see) step(key0, stage, there, turn, edge_tile);
      stage ^= STAGEB;
      turn = after;
    };
    auto whole = [&]() {
      bool all = next.ks[0] >= 0.f;
#pragma unroll
      for (int n = 1; n < NB; ++n) all = all && next.ks[n] >= 0.f;
      return all;
    };
    int key0 = k_first;
    for (; key0 + T <= k_end && key0 + T <= least && whole(); key0 += T) pass(key0, std::false_type{});
    for (; key0 < k_end; key0 += T) pass(key0, std::true_type{});
    at_turn = {stage, turn};

#pragma unroll
    for (int j = 0; j < QT; ++j) {
      const float sum = xquad_sum(l[j]);
      const int r = row0 + 16 * j + c16;
      if (r >= q_rows.rows) continue;
      const int i = divide(r, p.by_group), h = hk * p.group + r - i * p.group;
      if (slot >= 0) {
        const int64_t w = (int64_t)slot * BLOCK + r - rb * BLOCK;
#pragma unroll
        for (int d = 0; d < DT16; ++d)  // a row that saw no key is zeros, whatever values that are no numbers left in o
          *reinterpret_cast<floatx4*>(p.ws_o + w * D + 16 * d + 4 * g) = sum == 0.f ? (floatx4){0.f, 0.f, 0.f, 0.f} : o[d][j];
        if (g == 0) {
          // the sum's sign tells what the reference is: a score has a negative one
          const Reference r = Reference::of<Tag>(m[j], off[j]);
          p.ws_ml[2 * w] = m[j] == FA_NEG_INF ? FA_NEG_INF : r.at;
          p.ws_ml[2 * w + 1] = r.score ? -sum : sum;
        }
      } else {
        const float inv = 1.f / sum;
        uint16_t* dst = p.o + b * p.so[0] + h * p.so[1] + i * p.so[2] + 4 * g;
#pragma unroll
        for (int d = 0; d < DT16; ++d)
          *reinterpret_cast<u32x2*>(dst + 16 * d) =
              sum == 0.f ? (u32x2){0u, 0u}
                         : (u32x2){E::pack2(o[d][j][0] * inv, o[d][j][1] * inv), E::pack2(o[d][j][2] * inv, o[d][j][3] * inv)};
        if (g == 0 && p.lse != nullptr)
          p.lse[b * p.sl[0] + h * p.sl[1] + i * p.sl[2]] =
              sum == 0.f ? FA_NEG_INF : (__builtin_amdgcn_logf(sum) - off[j]) * 0.6931471805599453f;
      }
    }
  }
};

// Joins the parts of a row block: weights exp2 of their references' distance to the largest, of the unnormalised sums. A
// wave takes a row, D / 4 lanes a part's row; a workgroup kJoinRows rows of a block. About 700 parts of 64 KB (2 x 28 heads,
// 509 rows): 12.4 us, 3.9 TB/s.
constexpr int kJoinRows = 4;
template <typename Tag, int D, int BLOCK>
__device__ inline void join_parts(const Kv8AttendParams& p) {
  constexpr int LPS = D / 4, AT_ONCE = 64 / LPS, GROUPS = BLOCK / kJoinRows;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int block = (int)(blockIdx.x / GROUPS);  // hk, b, rb
  const int first = p.parts[2 * (int64_t)block], n = p.parts[2 * (int64_t)block + 1];
  if (n <= 1) return;
  const int pair = divide(block, p.by_blocks), rb = block - pair * p.row_blocks, hk = pair / p.B, b = pair % p.B;
  const int c4 = lane % LPS;
  for (int k = wave; k < kJoinRows; k += 4) {
    const int at = (int)(blockIdx.x % GROUPS) * kJoinRows + k, r = rb * BLOCK + at;
    if (r >= p.M * p.group) return;
    auto place = [&](int s) { return (int64_t)(s == 0 ? 2 * first + 1 : 2 * (first + s)) * BLOCK + at; };
    float m = FA_NEG_INF, sum = 0.f;  // m: the largest reference
    floatx4 o = (floatx4){0.f, 0.f, 0.f, 0.f};
    uint32_t signs = 0;
    for (int s = lane / LPS; s < n; s += AT_ONCE) {
      const u32x2 part = *reinterpret_cast<const u32x2*>(p.ws_ml + 2 * place(s));
      m = fmaxf(m, __uint_as_float(part[0]));
      signs |= part[1];
    }
    auto add = [&](int64_t w, float f) {
      const floatx4 x = *reinterpret_cast<const floatx4*>(p.ws_o + w * D + 4 * c4);
      sum = fmaf(f, fabsf(p.ws_ml[2 * w + 1]), sum);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = fmaf(f, x[j], o[j]);
    };
    if (__builtin_expect(__any((int)signs < 0), 0)) {
      // A part's reference is a score (rare). The largest is looked for by what they are about, by every lane in all parts.
      Reference top = {0.f, false};
      m = FA_NEG_INF;
      auto reference = [&](int s) {
        return Reference{p.ws_ml[2 * place(s)], __builtin_signbitf(p.ws_ml[2 * place(s) + 1]) != 0};
      };
      for (int s = 0; s < n; ++s) {
        const Reference r = reference(s);
        const float about = r.score ? r.at * p.c : r.at;
        if (about > m) top = r;
        m = fmaxf(m, about);
      }
      for (int s = lane / LPS; s < n; s += AT_ONCE) {
        const Reference r = reference(s);
        add(place(s), r.at == FA_NEG_INF ? 0.f : fast_exp2(r.less(top, p.c)));
      }
    } else {
      const float base = m == FA_NEG_INF ? 0.f : m;
#pragma unroll 2
      for (int s = lane / LPS; s < n; s += AT_ONCE) add(place(s), fast_exp2(p.ws_ml[2 * place(s)] - base));
    }
#pragma unroll
    for (int x = LPS; x < 64; x *= 2) {  // the wave's lane groups
      const float mo = __shfl_xor(m, x, 64), so = __shfl_xor(sum, x, 64);
      const float both = fmaxf(m, mo), ref = both == FA_NEG_INF ? 0.f : both;
      const float f = fast_exp2(m - ref), fo = fast_exp2(mo - ref);
      sum = f * sum + fo * so;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = f * o[j] + fo * __shfl_xor(o[j], x, 64);
      m = both;
    }
    if (lane >= LPS) continue;
    const int i = divide(r, p.by_group), h = hk * p.group + r - i * p.group;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<u32x2*>(p.o + b * p.so[0] + h * p.so[1] + i * p.so[2] + 4 * c4) =
        (u32x2){DT<Tag>::pack2(o[0] * inv, o[1] * inv), DT<Tag>::pack2(o[2] * inv, o[3] * inv)};
    if (c4 == 0 && p.lse != nullptr)
      p.lse[b * p.sl[0] + h * p.sl[1] + i * p.sl[2]] =
          sum == 0.f ? FA_NEG_INF : (m + __builtin_amdgcn_logf(sum) - lag_bias<Tag>()) * 0.6931471805599453f;
  }
}

template <typename Tag, int D>
__global__ __launch_bounds__(256) void kv8_join_kernel(Kv8AttendParams p) {
  join_parts<Tag, D, Kv8Chunk<Tag, D>::BLOCK>(p);
}

// Workgroups to a CU. At D = 64 the third costs 4 spilled registers (5 in fp16), and 1024 rows against 16k keys twice took
// 207 us where two workgroups took 221 (192 now).
template <int D>
constexpr int chunk8_waves() {
  return D == 64 ? 3 : 2;
}
template <typename Tag, int D>
__global__ __launch_bounds__(256, (chunk8_waves<D>())) void kv8_chunk_kernel(Kv8AttendParams p) {
  __shared__ __align__(1024) char smem[Kv8Chunk<Tag, D>::SMEM];
  __shared__ uint32_t flags[3][2];
  Kv8Chunk<Tag, D>::run(p, smem, flags);
}

template <typename Tag, int D, int WPR>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 256) void kv8_merge_kernel(Kv8AttendParams p) {
  merge_splits<Tag, D, WPR>(p, p.c);
}

#define KV8_ENTRY(TAG, DTYPE, D)                                                                            \
  {DTYPE, D, (const void*)&kv8_append_kernel<TAG, D>,                                                       \
   {(const void*)&kv8_merge_kernel<TAG, D, 1>, (const void*)&kv8_merge_kernel<TAG, D, 4>,                   \
    (const void*)&kv8_merge_kernel<TAG, D, 16>},                                                            \
   {(const void*)&kv8_attend_kernel<TAG, D, 1>, attend_two_tiles<TAG, D>(), (const void*)&kv8_chunk_kernel<TAG, D>}, \
   (const void*)&kv8_join_kernel<TAG, D>,                                                                   \
   {attend8_waves<D, 1>(), attend8_waves<D, 2>(), chunk8_waves<D>()},                                       \
   Kv8Chunk<TAG, D>::BLOCK, kJoinRows}

static const Kv8KernelEntry kKv8Entries[] = {
    KV8_ENTRY(f16_t, FA_DTYPE_F16, 64),   KV8_ENTRY(f16_t, FA_DTYPE_F16, 128),   KV8_ENTRY(f16_t, FA_DTYPE_F16, 256),
    KV8_ENTRY(bf16_t, FA_DTYPE_BF16, 64), KV8_ENTRY(bf16_t, FA_DTYPE_BF16, 128), KV8_ENTRY(bf16_t, FA_DTYPE_BF16, 256),
};

const Kv8KernelEntry* kv8_registry(int* count) {
  *count = (int)(sizeof(kKv8Entries) / sizeof(kKv8Entries[0]));
  return kKv8Entries;
}

}  // namespace fa
