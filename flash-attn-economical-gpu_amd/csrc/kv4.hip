// 4-bit key/value cache for gfx950: append of new rows, and attention over the cache.
//
// Format. A cached row of D channels is D / 32 blocks; a block is one scale byte e, standing for 2^(e - 127),
// and 32 codes of 4 bits (sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6). gfx950
// converts such codes to fp16 or bf16, scale included, two to an instruction (v_cvt_scalef32_pk_*_fp4), so
// reading the cache costs half an instruction per channel and the products stay 16-bit MFMAs on exact values.
// e = 255 is a block that held an infinity or NaN: all of it reads as NaN.
#include <type_traits>

#include "fa_common.h"
#include "fa_kernels.h"
#include "../../include/fa_gfx950.h"

namespace fa {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

template <typename Tag>
struct Fp4;
template <>
struct Fp4<f16_t> {
  // Range of scale bytes: the smallest and largest values, 0.5 and 6 times 2^(e - 127), are numbers of the type.
  static constexpr int kFloor = 104, kCeil = 140;
  static constexpr uint32_t kInfBits = 0x7c00u;
  // log2 of what P is scaled by on its way to fp16: weights down to 2^-29 keep all their bits.
  static constexpr float kPBias = 15.f;
  template <int SEL>
  __device__ static inline uint32_t encode(uint32_t old, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(half2_t, pair), scale, SEL);
  }
  template <int SEL>
  __device__ static inline uint32_t decode(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
  }
};
template <>
struct Fp4<bf16_t> {
  static constexpr int kFloor = 2, kCeil = 252;
  static constexpr uint32_t kInfBits = 0x7f80u;
  static constexpr float kPBias = 0.f;
  template <int SEL>
  __device__ static inline uint32_t encode(uint32_t old, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2_t, pair), scale, SEL);
  }
  template <int SEL>
  __device__ static inline uint32_t decode(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
  }
};

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

// Eight codes (a dword) to eight 16-bit values.
template <typename Tag>
__device__ inline u32x4 decode8(uint32_t codes, float scale) {
  return (u32x4){Fp4<Tag>::template decode<0>(codes, scale), Fp4<Tag>::template decode<1>(codes, scale),
                 Fp4<Tag>::template decode<2>(codes, scale), Fp4<Tag>::template decode<3>(codes, scale)};
}

// Append: a lane takes 8 channels, four neighbouring lanes a block. The scale puts the block's largest
// magnitude in [3.5, 7) steps: rounding to nearest reaches 6 from there with an error of at most one step,
// where a power below would clip 7 to 6 or a power above spend the top codes. Scale choice and conversion use
// integer compares and exact scalings only, so the result does not depend on the arithmetic of the host that
// checks it. Bound by memory (2 bytes in and 17/32 out per channel, 2 more with the values): 4 prompts of 2-4k tokens,
// 8 heads of 128, values returned, 136 MB in 26 us (5.3 TB/s; a copy of 4 GiB reaches 4.7); one token for 32
// sequences 4 us, a launch.
template <typename Tag>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4AppendParams p) {
  const int lpr = p.D / 8;
  const int64_t total = (int64_t)p.B * p.Hkv * p.rows * lpr;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const bool is_v = blockIdx.y != 0;
  if (id >= total) return;  // whole rows, so whole blocks, leave together
  const int part = (int)(id % lpr);
  const int64_t rest = id / lpr;
  // consecutive rows of a projection output [B, S, H, D] are its heads
  const int h = (int)(rest % p.Hkv);
  const int64_t br = rest / p.Hkv;
  const int row = (int)(br % p.rows), b = (int)(br / p.rows);
  const int64_t* st = is_v ? p.sv : p.sk;
  const uint16_t* src = (is_v ? p.v : p.k) + b * st[0] + h * st[1] + row * st[2] + part * 8;
  const int count = p.count != nullptr ? p.count[b] : p.rows;
  const int64_t at = (int64_t)p.start[b] + row;
  const bool live = row < count && at >= 0 && at < p.capacity;
  uint16_t* out = is_v ? p.v_values : p.k_values;
  u32x4 back = (u32x4){0, 0, 0, 0};
  if (live) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(src);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = x[j] & 0x7fffu, hi = (x[j] >> 16) & 0x7fffu;
      top = top > lo ? top : lo;
      top = top > hi ? top : hi;
    }
#pragma unroll
    for (int s = 1; s < 4; s *= 2) {
      const uint32_t o = __shfl_xor(top, s, 64);
      top = top > o ? top : o;
    }
    uint32_t e, codes = 0;
    if (top >= Fp4<Tag>::kInfBits) {
      e = 255;
    } else {
      const int up = (int)((__float_as_uint(DT<Tag>::to_float((uint16_t)top)) + 0x200000u) >> 23) - 2;
      e = (uint32_t)(up < Fp4<Tag>::kFloor ? Fp4<Tag>::kFloor : (up > Fp4<Tag>::kCeil ? Fp4<Tag>::kCeil : up));
      const float scale = scale_of(e);
      codes = Fp4<Tag>::template encode<0>(codes, x[0], scale);
      codes = Fp4<Tag>::template encode<1>(codes, x[1], scale);
      codes = Fp4<Tag>::template encode<2>(codes, x[2], scale);
      codes = Fp4<Tag>::template encode<3>(codes, x[3], scale);
    }
    uint8_t* cd = (is_v ? p.v_codes : p.k_codes) + b * p.code_stride[0] + h * p.code_stride[1] + at * (p.D / 2);
    uint8_t* sc = (is_v ? p.v_scales : p.k_scales) + b * p.scale_stride[0] + h * p.scale_stride[1] + at * (p.D / 32);
    *reinterpret_cast<uint32_t*>(cd + part * 4) = codes;
    if (part % 4 == 0) sc[part / 4] = (uint8_t)e;
    if (out != nullptr) back = decode8<Tag>(codes, scale_of(e));
  }
  if (out != nullptr) {
    const int64_t* so = is_v ? p.svv : p.skv;
    *reinterpret_cast<u32x4*>(out + b * so[0] + h * so[1] + row * so[2] + part * 8) = back;
  }
}

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
constexpr int kAllTiles = KV4_MAX_CAPACITY / 32;  // of the largest cache: the share where nothing is split
static_assert(KV4_MAX_CAPACITY % 32 == 0 && (uint64_t)kAllTiles * 64 <= 0xffffffffu,
              "64 sequences of whole tiles are summed in 32 bits");

struct Split {
  int b, index;     // sequence, and which of its splits (b < 0: a slot that no split has)
  int first, used;  // the sequence's first slot and number of splits
  int per;          // tiles of a split
};

// The split of a slot (slot >= 0), or of sequence b (slot < 0: only first, used and per are set).
__device__ inline Split find_split(const Kv4AttendParams& p, int slot, int b) {
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

// Attention over the cache. A wave holds 16 R query rows (columns of every product) and walks 32-key tiles:
//   S^T = K Q^T     A = K rows: lane (key, quarter of D) reads its quarter row and converts it in place
//   O^T += V^T P^T  A = V^T: lane (channels, 8 keys) reads the keys' codes of its D / 16 channels, converts, and
//                   regroups them by channel with byte permutes; P^T is S^T's accumulator as it stands
// so nothing passes through LDS but the waves' sums at the end. About 170 vector instructions a wave and tile at
// D = 128, 100 of them conversion, take some 40% of the vector slots at the rate memory delivers; two tiles in flight per wave and two to four waves per SIMD cover the
// latency. 8 sequences of 16-32k tokens, 8 heads of 128: 223 MB in 46 us (4.8 TB/s) and 6 us for the join; one
// sequence of 8k: 7.2 + 5 us, launch and dependent-load latencies. Query rows are (position, head of the group):
// row r is head r % group at position r / group, and a workgroup's rows share its kv head's cache.
// The four waves hold the same rows (single tokens, short drafts) and take turns at the tiles.
template <typename Tag, int D, int R>
struct Kv4Attend {
  static constexpr int WAVES = 4;
  static constexpr int KS = D / 32;   // k = 32 steps over D
  static constexpr int CPL = D / 16;  // channels of V per lane
  static constexpr int SB = D / 32;   // scale bytes of a row
  static constexpr int CB = D / 2;    // code bytes of a row
  static constexpr int KW = D / 32;   // dwords of K codes per lane and key
  static constexpr int VS = D == 64 ? 4 : 8;  // dwords of V scales per lane and tile
  typedef DT<Tag> E;

  struct Tile {  // one lane's share of a 32-key tile, as stored
    uint32_t k[2][KW];
    uint32_t ks[2];
    uint32_t v[8][CPL >= 8 ? CPL / 8 : 1];
    uint32_t vs[VS];
  };

  // Keys of a lane's k-slots in the second product: slot i is key 4 g + (i & 3) + 16 (i >> 2).
  __device__ static inline void load(Tile& t, const uint8_t* kc, const uint8_t* ksc, const uint8_t* vc,
                                     const uint8_t* vsc, int key0, int lane) {
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t key = key0 + 16 * i + r;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(kc + key * CB + g * (D / 8));
#pragma unroll
      for (int w = 0; w < KW; ++w) t.k[i][w] = src[w];
      if constexpr (D == 256)
        t.ks[i] = *reinterpret_cast<const uint16_t*>(ksc + key * SB + 2 * g);
      else
        t.ks[i] = ksc[key * SB + (D == 64 ? g / 2 : g)];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t key = key0 + 4 * g + (i & 3) + 16 * (i >> 2);
      const uint8_t* src = vc + key * CB + r * (CPL / 2);
      if constexpr (CPL == 4) {
        t.v[i][0] = *reinterpret_cast<const uint16_t*>(src);
      } else {
#pragma unroll
        for (int w = 0; w < CPL / 8; ++w) t.v[i][w] = reinterpret_cast<const uint32_t*>(src)[w];
      }
      if constexpr (D == 256) t.vs[i] = vsc[key * SB + r * CPL / 32];
    }
    if constexpr (D != 256) {  // all scales of four neighbouring keys in one load; scale() takes the lane's block
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t* src = vsc + (int64_t)(key0 + 4 * g + 16 * i) * SB;
        if constexpr (D == 64) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(src);
          t.vs[2 * i] = x[0];
          t.vs[2 * i + 1] = x[1];
        } else {
          const u32x4 x = *reinterpret_cast<const u32x4*>(src);
#pragma unroll
          for (int j = 0; j < 4; ++j) t.vs[4 * i + j] = x[j];
        }
      }
    }
  }
  // V's scale of the lane's i-th key
  __device__ static inline float v_scale(const Tile& t, int i, int lane) {
    const uint32_t blk = (uint32_t)(lane & 15) * CPL / 32;
    if constexpr (D == 256) return scale_of(t.vs[i]);
    if constexpr (D == 128) return scale_of((t.vs[i] >> (8 * blk)) & 255u);
    return scale_of((t.vs[i / 2] >> (8 * blk + 16 * (i & 1))) & 255u);
  }

  struct State {
    floatx4 o[CPL][R];
    float m[R], l[R];
  };

  // The n-th key's values, of the blocks marked in `bad` only, times P: a product of its own, whose result only the
  // rows that see the key take.
  __device__ static inline void add_alone(State& s, const Tile& t, const float (&vs)[8], const u32x4 (&pb)[R], uint32_t bad,
                                          int n, int key0, const int (&see)[R], int lane) {
    const int slot = (n & 3) + 4 * (n >> 4);
    const bool mine = lane >> 4 == ((n >> 2) & 3) && (bad >> slot & 1u) != 0;
    if (!__any(mine)) return;
    uint32_t code[CPL >= 8 ? CPL / 8 : 1] = {};
    float scale = 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i == slot) {
        scale = vs[i];
#pragma unroll
        for (int w = 0; w < (CPL >= 8 ? CPL / 8 : 1); ++w) code[w] = t.v[i][w];
      }
    auto pair = [&](auto jc) {
      constexpr int j = decltype(jc)::value;
      const uint32_t x = mine ? Fp4<Tag>::template decode<j % 4>(code[j / 4], scale) : 0u;
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

  // One tile: keys [key0, key0 + 32), of which row rt sees those below see[rt] (a lane's own row). `unseen`: a row
  // before count does not see all of the sequence's keys among them.
  template <bool EDGE>
  __device__ static inline void step(State& s, const u32x4 (&qf)[R][KS], Tile& t, int key0, const int (&see)[R],
                                     int keys, bool unseen, float c, int lane) {
    const int g = lane >> 4;
    floatx4 x[2][R];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int rt = 0; rt < R; ++rt) x[i][rt] = (floatx4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const float scale = scale_of(D == 256 ? (t.ks[i] >> (8 * (k >> 2))) & 255u : t.ks[i]);
        const u32x4 a = decode8<Tag>(t.k[i][k], scale);
#pragma unroll
        for (int rt = 0; rt < R; ++rt) x[i][rt] = E::mfma16(a, qf[rt][k], x[i][rt]);
      }
    }
    u32x4 pb[R];
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      if constexpr (EDGE) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key0 + 16 * i + 4 * g + r >= see[rt]) x[i][rt][r] = FA_NEG_INF;
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
      const float off = Fp4<Tag>::kPBias - (s.m[rt] == FA_NEG_INF ? 0.f : s.m[rt] * c);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[i][rt][r] = fast_exp2(fmaf(x[i][rt][r], c, off));
          s.l[rt] += x[i][rt][r];
        }
      pb[rt] = (u32x4){E::pack2(x[0][rt][0], x[0][rt][1]), E::pack2(x[0][rt][2], x[0][rt][3]),
                       E::pack2(x[1][rt][0], x[1][rt][1]), E::pack2(x[1][rt][2], x[1][rt][3])};
    }
    float vs[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      vs[i] = v_scale(t, i, lane);
      if constexpr (EDGE) {  // rows behind the last key may hold anything, NaN too: they read as zeros
        if (key0 + 4 * g + (i & 3) + 16 * (i >> 2) >= keys) {
          vs[i] = 1.f;
#pragma unroll
          for (int w = 0; w < (CPL >= 8 ? CPL / 8 : 1); ++w) t.v[i][w] = 0;
        }
      }
    }
    if constexpr (EDGE) {
      // A block that is NaN, or whose scale takes it past the type, would be 0 x NaN to the rows that do not see it.
      // Such blocks (rare) leave the tile's product and are added key by key.
      uint32_t bad = 0;
      if (unseen) {
#pragma unroll
        for (int i = 0; i < 8; ++i) bad |= (vs[i] > scale_of(Fp4<Tag>::kCeil) ? 1u : 0u) << i;
      }
      if (__builtin_expect(__any(bad != 0), 0)) {
#pragma unroll 1
        for (int n = 0; n < 32; ++n) add_alone(s, t, vs, pb, bad, n, key0, see, lane);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (bad >> i & 1u) {
            vs[i] = 1.f;
#pragma unroll
            for (int w = 0; w < (CPL >= 8 ? CPL / 8 : 1); ++w) t.v[i][w] = 0;
          }
      }
    }
    // channels 2 j and 2 j + 1 of the lane's CPL: byte j of a key's codes
    auto pair = [&](auto jc) {
      constexpr int j = decltype(jc)::value;
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = Fp4<Tag>::template decode<j % 4>(t.v[i][j / 4], vs[i]);
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
  }

  template <int N, int J = 0, typename F>
  __device__ static inline void for_each(F& f) {
    if constexpr (J < N) {
      f(std::integral_constant<int, J>{});
      for_each<N, J + 1>(f);
    }
  }

  // N channels N at .. of row r, whose maximum and sum are m and l. A row that saw no key (l = 0) is zeros, whatever its
  // products with values that are no numbers left in o.
  template <int N>
  __device__ static inline void store_row(const Kv4AttendParams& p, int b, int hk, int slot, int r, const float (&o)[N],
                                          float m, float l, int at) {
    const int i = r / p.group, h = hk * p.group + r % p.group;
    if (p.splits > 1) {
      const int64_t w = ((int64_t)slot * p.H + h) * p.M + i;
      float* dst = p.ws_o + w * D + at * N;
#pragma unroll
      for (int j = 0; j < N; j += 4)
        *reinterpret_cast<floatx4*>(dst + j) = l == 0.f ? (floatx4){0.f, 0.f, 0.f, 0.f} : (floatx4){o[j], o[j + 1], o[j + 2], o[j + 3]};
      if (at == 0) {
        p.ws_ml[2 * w] = m * p.c;
        p.ws_ml[2 * w + 1] = l;
      }
    } else {
      const float inv = 1.f / l;
      uint16_t* dst = p.o + b * p.so[0] + h * p.so[1] + i * p.so[2] + at * N;
#pragma unroll
      for (int j = 0; j < N; j += 4)
        *reinterpret_cast<u32x2*>(dst + j) = l == 0.f ? (u32x2){0u, 0u} : (u32x2){E::pack2(o[j] * inv, o[j + 1] * inv), E::pack2(o[j + 2] * inv, o[j + 3] * inv)};
      if (at == 0 && p.lse != nullptr)
        p.lse[b * p.sl[0] + h * p.sl[1] + i * p.sl[2]] =
            l == 0.f ? FA_NEG_INF : (m * p.c + __builtin_amdgcn_logf(l) - Fp4<Tag>::kPBias) * 0.6931471805599453f;
    }
  }

  __device__ static void run(const Kv4AttendParams& p, float* smem) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    // row blocks innermost: those of one split share its tiles in L2
    const int rb = id % p.row_blocks;
    id /= p.row_blocks;
    const int slot = id % p.slots, hk = id / p.slots;
    const Split part = find_split(p, slot, 0);
    const int b = __builtin_amdgcn_readfirstlane(part.b);
    if (b < 0) return;
    const int rows = p.M * p.group;
    const int row0 = rb * 16 * R;
    const int keys = visible_keys(p.start, p.count, b, p.M, p.capacity);
    const int count = p.count != nullptr ? p.count[b] : p.M;
    const int64_t start = p.start[b];

    int see[R];  // keys that the lane's row sees
    u32x4 qf[R][KS];
    State s;
    const int wave_top = row0 + 16 * R <= rows ? row0 + 16 * R - 1 : rows - 1;  // the wave's last row sees most
    int wave_see = 0;
    if (row0 < rows) {
      const int64_t e = p.causal ? start + wave_top / p.group + 1 : keys;
      wave_see = (int)(e < 0 ? 0 : (e > keys ? keys : e));
    }
    int least = wave_see;   // keys that every row of the wave sees
    int live_least = 0x7fffffff;  // and those that every row before count sees
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      const int r = row0 + 16 * rt + c16;
      const int i = r / p.group;
      const bool live = r < rows && i < count;
      const int64_t e = p.causal ? start + i + 1 : keys;
      see[rt] = !live || e < 0 ? 0 : (int)(e > keys ? keys : e);
      const uint16_t* q = p.q + b * p.sq[0] + (int64_t)(hk * p.group + (r < rows ? r % p.group : 0)) * p.sq[1] +
                          (int64_t)(r < rows ? i : 0) * p.sq[2] + g * (D / 4);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qf[rt][k] = (u32x4){0, 0, 0, 0};
        if (live) qf[rt][k] = *reinterpret_cast<const u32x4*>(q + 8 * k);
      }
      s.m[rt] = FA_NEG_INF;
      s.l[rt] = 0.f;
#pragma unroll
      for (int d = 0; d < CPL; ++d) s.o[d][rt] = (floatx4){0.f, 0.f, 0.f, 0.f};
    }
    if (row0 < rows) {
      const int64_t e = p.causal ? start + row0 / p.group + 1 : keys;
      const int64_t low = e < 0 ? 0 : (e > keys ? keys : e);
      least = wave_top / p.group < count && row0 + 16 * R <= rows ? (int)low : 0;
      if (row0 / p.group < count) live_least = (int)low;
    }
    const int tiles = (wave_see + 31) / 32;
    const int per = __builtin_amdgcn_readfirstlane(part.per);
    int t0 = __builtin_amdgcn_readfirstlane(part.index) * per, t1 = t0 + per < tiles ? t0 + per : tiles;
    const uint8_t* kc = p.k_codes + b * p.code_stride[0] + hk * p.code_stride[1];
    const uint8_t* vc = p.v_codes + b * p.code_stride[0] + hk * p.code_stride[1];
    const uint8_t* ks = p.k_scales + b * p.scale_stride[0] + hk * p.scale_stride[1];
    const uint8_t* vs = p.v_scales + b * p.scale_stride[0] + hk * p.scale_stride[1];
    t0 += wave;
    // in vector registers: with scalar branches the allocator spills a hundred bytes inside the loop
    asm volatile("" : "+v"(t1), "+v"(least));
    // two tiles in flight
    Tile even, odd;
    auto fetch = [&](Tile& x, int t) {
      if (t < t1) load(x, kc, ks, vc, vs, t * 32, lane);
    };
    auto use = [&](Tile& x, int t) {
      if (t * 32 + 32 <= least) step<false>(s, qf, x, t * 32, see, keys, false, p.c, lane);
      else step<true>(s, qf, x, t * 32, see, keys, (t * 32 + 32 < keys ? t * 32 + 32 : keys) > live_least, p.c, lane);
      fetch(x, t + 2 * WAVES);
    };
    fetch(even, t0);
    fetch(odd, t0 + WAVES);
    for (int t = t0; t < t1; t += 2 * WAVES) {
      use(even, t);
      if (t + WAVES < t1) use(odd, t + WAVES);
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
      if (r < rows) store_row<CPL>(p, b, hk, slot, r, o, m, sum, c16);
      __syncthreads();
    }
  }
};

// Waves per SIMD: what the registers of two tiles in flight, Q and O allow.
template <int D, int R>
constexpr int attend_waves() {
  return D == 64 ? (R == 1 ? 4 : 3) : (D == 128 ? (R == 1 ? 3 : 2) : (R == 1 ? 2 : 1));
}
template <typename Tag, int D, int R>
__global__ __launch_bounds__(256, (attend_waves<D, R>())) void kv4_attend_kernel(Kv4AttendParams p) {
  __shared__ __align__(16) float smem[4 * 16 * (D + 4)];
  Kv4Attend<Tag, D, R>::run(p, smem);
}

// Chunks of a prompt: more than 32 query rows to a kv head. Here the conversion would cost each wave more than its
// products if it did it for itself (455 TFLOP/s at 32 rows a wave), so the workgroup's four waves, of 32 rows each,
// share it: a tile's codes are loaded a tile ahead, 32 channels of a row to a thread, converted once into 16-bit
// rows in LDS (two stages, one barrier a tile), and both products read their fragments there, V's by the
// transposing read. S^T = K Q^T and O^T = V^T P^T as above. Bound by the softmax's vector work beside the MFMAs (216
// vector instructions, 32 of them exponentials, to 64 MFMAs a wave and tile at D = 128): 970 TFLOP/s where the grid
// fills the chip (1024 rows over 32k keys, 32/8 heads), 610 with 448 workgroups for 512 places (509 and 382 rows over 16k
// and 12k, 28/4 heads). 56 of those 448 hold no row before count: their zeros are right, but they walk the keys for
// nothing, and rows behind count cost as much as rows before it. 32-key tiles at D = 128 and converting a tile ahead were 5 to 7% slower.
template <typename Tag, int D>
struct Kv4Chunk {
  using L = LdsRows<D>;
  typedef DT<Tag> E;
  static constexpr int WAVES = 4, QT = D == 256 ? 1 : 2;  // 16-row tiles of queries per wave
  static constexpr int T = D == 256 ? 32 : 64;  // keys of a tile
  static constexpr int KT = T / 16, KS = D / 32, DT16 = D / 16, SB = D / 32;
  static constexpr int BLOCK = WAVES * QT * 16;
  static constexpr int TILEB = T * L::ROWB, STAGEB = 2 * TILEB;
  static constexpr int SMEM = 2 * STAGEB;
  static constexpr int UNITS = T * SB;              // 32-channel units of one matrix' tile
  static constexpr int PER = 2 * UNITS / (WAVES * 64);  // units per thread: one (D = 64: K or V), else one of each
  static_assert(PER == 1 || PER == 2, "units");

  struct Codes {
    u32x4 c[PER];
    uint32_t e[PER];
  };

  __device__ static void run(const Kv4AttendParams& p, char* smem) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    const int rb = id % p.row_blocks;
    id /= p.row_blocks;
    const int slot = id % p.slots, hk = id / p.slots;
    const Split part = find_split(p, slot, 0);
    const int b = __builtin_amdgcn_readfirstlane(part.b);
    if (b < 0) return;
    const int rows = p.M * p.group, row0 = rb * BLOCK + wave * QT * 16;
    const int keys = visible_keys(p.start, p.count, b, p.M, p.capacity);
    const int count = p.count != nullptr ? p.count[b] : p.M;
    const int64_t start = p.start[b];
    auto seen = [&](int row) {  // keys that a live row sees
      const int64_t e = p.causal ? start + row / p.group + 1 : keys;
      return (int)(e < 0 ? 0 : (e > keys ? keys : e));
    };
    auto last_live = [&](int first, int n) {  // the last of n rows that exists
      return first + n <= rows ? first + n - 1 : rows - 1;
    };
    const int block_see = seen(last_live(rb * BLOCK, BLOCK));
    const int wave_see = __builtin_amdgcn_readfirstlane(row0 < rows ? seen(last_live(row0, QT * 16)) : 0);
    const bool whole = row0 + QT * 16 <= rows && (row0 + QT * 16 - 1) / p.group < count;
    const int least = __builtin_amdgcn_readfirstlane(whole ? seen(row0) : 0);  // keys that every row of the wave sees

    int see[QT];
    u32x4 qf[QT][KS];
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      const int r = row0 + 16 * j + c16, i = r / p.group;
      const bool live = r < rows && i < count;
      see[j] = live ? seen(r) : 0;
      const uint16_t* q = p.q + b * p.sq[0] + (int64_t)(hk * p.group + (live ? r % p.group : 0)) * p.sq[1] +
                          (int64_t)(live ? i : 0) * p.sq[2] + 8 * g;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qf[j][k] = (u32x4){0, 0, 0, 0};
        if (live) qf[j][k] = *reinterpret_cast<const u32x4*>(q + 32 * k);
      }
    }
    floatx4 o[DT16][QT];
    float m[QT], l[QT];
#pragma unroll
    for (int j = 0; j < QT; ++j) {
      m[j] = FA_NEG_INF;
      l[j] = 0.f;
#pragma unroll
      for (int d = 0; d < DT16; ++d) o[d][j] = (floatx4){0.f, 0.f, 0.f, 0.f};
    }

    // the split's keys, in tiles of T (its share is in tiles of 32)
    const int64_t per = (int64_t)__builtin_amdgcn_readfirstlane(part.per) * 32;
    const int64_t k_first = __builtin_amdgcn_readfirstlane(part.index) * per;
    const int k_end = __builtin_amdgcn_readfirstlane((int)(k_first + per < block_see ? k_first + per : block_see));
#pragma unroll
    for (int j = 0; j < QT; ++j) see[j] = see[j] < k_end ? see[j] : k_end;  // the next split may begin inside a tile
    // of the split's keys, those that every row before count sees
    const int live_least = __builtin_amdgcn_readfirstlane(
        row0 < rows && row0 / p.group < count ? (seen(row0) < k_end ? seen(row0) : k_end) : 0x7fffffff);
    const uint8_t* kc = p.k_codes + b * p.code_stride[0] + hk * p.code_stride[1];
    const uint8_t* vc = p.v_codes + b * p.code_stride[0] + hk * p.code_stride[1];
    const uint8_t* ksc = p.k_scales + b * p.scale_stride[0] + hk * p.scale_stride[1];
    const uint8_t* vsc = p.v_scales + b * p.scale_stride[0] + hk * p.scale_stride[1];
    // thread's unit u of the tile at key0: rows are dense, so units are too. Past the last visible key nothing is read,
    // and what stands there is zero: rows behind a sequence may hold anything.
    auto fetch = [&](Codes& x, int64_t key0) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const bool is_v = PER == 1 ? tid >= UNITS : i == 1;
        const int u = PER == 1 ? tid % UNITS : tid;
        x.c[i] = (u32x4){0, 0, 0, 0};
        x.e[i] = 127;
        if (key0 + u / SB < keys) {
          const int64_t at = key0 * SB + u;
          x.c[i] = *reinterpret_cast<const u32x4*>((is_v ? vc : kc) + at * 16);
          x.e[i] = (is_v ? vsc : ksc)[at];
        }
      }
    };
    auto convert = [&](const Codes& x, uint32_t stage) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const bool is_v = PER == 1 ? tid >= UNITS : i == 1;
        const int u = PER == 1 ? tid % UNITS : tid;
        const int row = u / SB, blk = u % SB;
        char* dst = smem + stage + (is_v ? TILEB : 0) + row * L::ROWB;
        const float scale = scale_of(x.e[i]);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<u32x4*>(dst + (((4 * blk + c) ^ L::swz(row)) << 4)) = decode8<Tag>(x.c[i][c], scale);
      }
    };
    const uint32_t ro = L::row_off(lane), to = L::tr_off(lane);
    auto step = [&](int key0, uint32_t stage, auto edge_tile) {
      constexpr bool EDGE = decltype(edge_tile)::value;
      const uint32_t rowb = ro + stage, colb = to + stage;
      // A block that is NaN or past the type would be 0 x NaN to the rows that do not see it: keys that have one (rare)
      // are left out of the tile's product and added one by one, to the rows that see them. Looked for in the few
      // tiles that a row before count does not see whole.
      uint64_t alone = 0;  // keys of the tile
      if (EDGE && (key0 + T < keys ? key0 + T : keys) > live_least) {
        bool bad = false;
        if (lane < T && key0 + lane < keys) {
          typedef uint8_t scales_t __attribute__((ext_vector_type(SB)));
          const scales_t e = *reinterpret_cast<const scales_t*>(vsc + (int64_t)(key0 + lane) * SB);
#pragma unroll
          for (int n = 0; n < SB; ++n) bad |= e[n] > Fp4<Tag>::kCeil;
        }
        alone = __ballot(bad);
      }
      // D = 64: all of K's fragments (32 registers) are asked for before the first product. Left to the compiler they came
      // one by one, each waited for: 214 against 205 us (512 rows over 16k keys, 28/4 heads).
      u32x4 ahead[KT][KS];
      if constexpr (D == 64) {
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
          for (int k = 0; k < KS; ++k) ahead[i][k] = L::frag(smem, rowb ^ (k << 6), i * 16 * L::ROWB);
        __builtin_amdgcn_sched_barrier(0);
      }
      floatx4 x[KT][QT];
#pragma unroll
      for (int i = 0; i < KT; ++i) {
#pragma unroll
        for (int j = 0; j < QT; ++j) x[i][j] = (floatx4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const u32x4 a = D == 64 ? ahead[i][k] : L::frag(smem, rowb ^ (k << 6), i * 16 * L::ROWB);
#pragma unroll
          for (int j = 0; j < QT; ++j) x[i][j] = E::mfma16(a, qf[j][k], x[i][j]);
        }
      }
      u32x4 pb[KT / 2][QT];
#pragma unroll
      for (int j = 0; j < QT; ++j) {
        float top = FA_NEG_INF;
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (EDGE && key0 + 16 * i + 4 * g + r >= see[j]) x[i][j][r] = FA_NEG_INF;
            top = larger(top, x[i][j][r]);
          }
        const float m_new = larger(m[j], row_max(top));
        if (__any(m_new > m[j])) {
          const float base = m_new == FA_NEG_INF ? 0.f : m_new;
          const float f = fast_exp2((m[j] - base) * p.c);
          l[j] *= f;
#pragma unroll
          for (int d = 0; d < DT16; ++d) o[d][j] *= f;
          m[j] = m_new;
        }
        const float off = Fp4<Tag>::kPBias - (m[j] == FA_NEG_INF ? 0.f : m[j] * p.c);
#pragma unroll
        for (int i = 0; i < KT; ++i) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[i][j][r] = fast_exp2(fmaf(x[i][j][r], p.c, off));
            l[j] += x[i][j][r];
          }
          pb[i / 2][j][2 * (i & 1)] = E::pack2(x[i][j][0], x[i][j][1]);
          pb[i / 2][j][2 * (i & 1) + 1] = E::pack2(x[i][j][2], x[i][j][3]);
        }
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
      __builtin_amdgcn_s_setprio(1);  // before a neighbour's softmax: 2 to 5%
#pragma unroll
      for (int d = 0; d < DT16; ++d)
#pragma unroll
        for (int i = 0; i < KT / 2; ++i) {
          u32x4 v = L::tfrag(smem, colb ^ (d << 5), TILEB + i * 32 * L::ROWB);
          if (EDGE && alone != 0) v &= ~lanes_of((uint32_t)(alone >> (32 * i)));
#pragma unroll
          for (int j = 0; j < QT; ++j) o[d][j] = E::mfma16(v, pb[i][j], o[d][j]);
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
    uint32_t stage = 0;
    // tiles that every row of the wave sees whole, then those on the diagonal or at the end: every wave makes the
    // same number of passes in all, for the barriers
    auto pass = [&](int64_t key0, auto edge_tile) {
      convert(next, stage);
      if (key0 + T < k_end) fetch(next, key0 + T);
      wait_vm_lds_barrier<63>();  // LDS writes only: the codes just asked for stay in flight
      if (key0 < wave_see) step((int)key0, stage, edge_tile);
      stage ^= STAGEB;
    };
    int64_t key0 = k_first;
    for (; key0 + T <= k_end && key0 + T <= least; key0 += T) pass(key0, std::false_type{});
    for (; key0 < k_end; key0 += T) pass(key0, std::true_type{});

#pragma unroll
    for (int j = 0; j < QT; ++j) {
      const float sum = xquad_sum(l[j]);
      const int r = row0 + 16 * j + c16;
      if (r >= rows) continue;
      const int i = r / p.group, h = hk * p.group + r % p.group;
      if (p.splits > 1) {
        const int64_t w = ((int64_t)slot * p.H + h) * p.M + i;
#pragma unroll
        for (int d = 0; d < DT16; ++d)  // a row that saw no key is zeros, whatever values that are no numbers left in o
          *reinterpret_cast<floatx4*>(p.ws_o + w * D + 16 * d + 4 * g) = sum == 0.f ? (floatx4){0.f, 0.f, 0.f, 0.f} : o[d][j];
        if (g == 0) {
          p.ws_ml[2 * w] = m[j] * p.c;
          p.ws_ml[2 * w + 1] = sum;
        }
      } else {
        const float inv = 1.f / sum;
        uint16_t* dst = p.o + b * p.so[0] + h * p.so[1] + i * p.so[2] + 4 * g;
#pragma unroll
        for (int d = 0; d < DT16; ++d)
          *reinterpret_cast<u32x2*>(dst + 16 * d) = sum == 0.f ? (u32x2){0u, 0u} :
              (u32x2){E::pack2(o[d][j][0] * inv, o[d][j][1] * inv), E::pack2(o[d][j][2] * inv, o[d][j][3] * inv)};
        if (g == 0 && p.lse != nullptr)
          p.lse[b * p.sl[0] + h * p.sl[1] + i * p.sl[2]] =
              sum == 0.f ? FA_NEG_INF : (m[j] * p.c + __builtin_amdgcn_logf(sum) - Fp4<Tag>::kPBias) * 0.6931471805599453f;
      }
    }
  }
};

template <typename Tag, int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void kv4_chunk_kernel(Kv4AttendParams p) {
  __shared__ __align__(1024) char smem[Kv4Chunk<Tag, D>::SMEM];
  Kv4Chunk<Tag, D>::run(p, smem);
}

// Joins the splits of a row: weights exp2(m_s - m) of the unnormalised partial sums. WPR waves take a row: one
// where rows are many and splits few, four or sixteen the other way round (single tokens over long caches). D / 4 lanes read one
// split's row, so a wave has 256 / D of them in flight at once, times the unrolling.
template <typename Tag, int D, int WPR>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 256) void kv4_merge_kernel(Kv4AttendParams p) {
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
      const float f = fast_exp2(p.ws_ml[2 * w] - base);
      const floatx4 x = *reinterpret_cast<const floatx4*>(p.ws_o + w * D + 4 * c4);
      sum = fmaf(f, p.ws_ml[2 * w + 1], sum);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = fmaf(f, x[j], o[j]);
    }
#pragma unroll
    for (int k = LPS; k < 64; k *= 2) {  // the wave's lane groups
      const float mo = __shfl_xor(m, k, 64), so = __shfl_xor(sum, k, 64);
      const float top = fmaxf(m, mo), ref = top == FA_NEG_INF ? 0.f : top;
      const float f = fast_exp2(m - ref), fo = fast_exp2(mo - ref);
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
        const float f = fast_exp2(part_ml[w][0] - ref);
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
          sum == 0.f ? FA_NEG_INF : (m + __builtin_amdgcn_logf(sum) - Fp4<Tag>::kPBias) * 0.6931471805599453f;
  }
}

#define KV4_ENTRY(TAG, DTYPE, D)                                                                                   \
  {DTYPE, D, (const void*)&kv4_append_kernel<TAG>,                                                                 \
   {(const void*)&kv4_merge_kernel<TAG, D, 1>, (const void*)&kv4_merge_kernel<TAG, D, 4>,                         \
    (const void*)&kv4_merge_kernel<TAG, D, 16>},                         \
   {(const void*)&kv4_attend_kernel<TAG, D, 1>, (const void*)&kv4_attend_kernel<TAG, D, 2>,            \
    (const void*)&kv4_chunk_kernel<TAG, D>},                                                                        \
   {attend_waves<D, 1>(), attend_waves<D, 2>(), 2}, Kv4Chunk<TAG, D>::BLOCK}

static const Kv4KernelEntry kKv4Entries[] = {
    KV4_ENTRY(f16_t, FA_DTYPE_F16, 64),   KV4_ENTRY(f16_t, FA_DTYPE_F16, 128),   KV4_ENTRY(f16_t, FA_DTYPE_F16, 256),
    KV4_ENTRY(bf16_t, FA_DTYPE_BF16, 64), KV4_ENTRY(bf16_t, FA_DTYPE_BF16, 128), KV4_ENTRY(bf16_t, FA_DTYPE_BF16, 256),
};

const Kv4KernelEntry* kv4_registry(int* count) {
  *count = (int)(sizeof(kKv4Entries) / sizeof(kKv4Entries[0]));
  return kKv4Entries;
}

}  // namespace fa
