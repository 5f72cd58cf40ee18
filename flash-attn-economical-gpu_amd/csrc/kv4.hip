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
// checks it. Bound by memory (2 bytes in and 17/32 out per channel, 2 more with the values).
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

// 32-key tiles of a split, the same for all splits of a sequence: at least kMinTiles, so short sequences in a
// large cache use few splits.
__device__ inline int tiles_per_split(int keys, int splits, int min_tiles) {
  const int tiles = (keys + 31) / 32;
  const int even = (tiles + splits - 1) / splits;
  return even > min_tiles ? even : min_tiles;
}

// Attention over the cache. A wave holds 16 R query rows (columns of every product) and walks 32-key tiles:
//   S^T = K Q^T     A = K rows: lane (key, quarter of D) reads its quarter row and converts it in place
//   O^T += V^T P^T  A = V^T: lane (channels, 8 keys) reads the keys' codes of its D / 16 channels, converts, and
//                   regroups them by channel with byte permutes; P^T is S^T's accumulator as it stands
// so nothing passes through LDS but the waves' sums at the end. Query rows are (position, head of the group):
// row r is head r % group at position r / group, and a workgroup's rows share its kv head's cache.
//   SHARED: the four waves hold the same rows and take turns at the tiles (single tokens, short drafts)
//   else:   each wave holds its own rows (chunks of a prompt)
template <typename Tag, int D, int R, bool SHARED>
struct Kv4Attend {
  static constexpr int WAVES = 4;
  static constexpr int KS = D / 32;   // k = 32 steps over D
  static constexpr int CPL = D / 16;  // channels of V per lane
  static constexpr int SB = D / 32;   // scale bytes of a row
  static constexpr int CB = D / 2;    // code bytes of a row
  static constexpr int KW = D / 32;   // dwords of K codes per lane and key
  typedef DT<Tag> E;

  struct Tile {  // one lane's share of a 32-key tile, as stored
    uint32_t k[2][KW];
    uint32_t ks[2];
    uint32_t v[8][CPL >= 8 ? CPL / 8 : 1];
    uint32_t vs[8];
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
      t.vs[i] = vsc[key * SB + r * CPL / 32];
    }
  }

  struct State {
    floatx4 o[CPL][R];
    float m[R], l[R];
  };

  // One tile: keys [key0, key0 + 32), of which row rt sees those below see[rt] (a lane's own row).
  template <bool EDGE>
  __device__ static inline void step(State& s, const u32x4 (&qf)[R][KS], Tile& t, int key0, const int (&see)[R],
                                     int keys, float c, int lane) {
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
      float top = fmaxf(fmaxf(fmaxf(x[0][rt][0], x[0][rt][1]), fmaxf(x[0][rt][2], x[0][rt][3])),
                        fmaxf(fmaxf(x[1][rt][0], x[1][rt][1]), fmaxf(x[1][rt][2], x[1][rt][3])));
      top = xquad_max(top);
      const float m_new = fmaxf(s.m[rt], top);
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
    if constexpr (EDGE) {  // rows behind the last key may hold anything, NaN too: they read as zeros
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (key0 + 4 * g + (i & 3) + 16 * (i >> 2) >= keys) {
          t.vs[i] = 127;
#pragma unroll
          for (int w = 0; w < (CPL >= 8 ? CPL / 8 : 1); ++w) t.v[i][w] = 0;
        }
    }
    // channels 2 j and 2 j + 1 of the lane's CPL: byte j of a key's codes
    auto pair = [&](auto jc) {
      constexpr int j = decltype(jc)::value;
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = Fp4<Tag>::template decode<j % 4>(t.v[i][j / 4], scale_of(t.vs[i]));
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

  // A lane's 4 CPL = D / 4 channels of row rt: channels (D / 4) g .. in order.
  __device__ static inline void store_row(const Kv4AttendParams& p, int b, int hk, int split, int r, const float* o,
                                          float m, float l, int g) {
    const int i = r / p.group, h = hk * p.group + r % p.group;
    if (p.splits > 1) {
      const int64_t row = ((int64_t)b * p.H + h) * p.M + i;
      const int64_t w = (int64_t)split * p.B * p.H * p.M + row;
      float* dst = p.ws_o + w * D + g * (D / 4);
#pragma unroll
      for (int j = 0; j < D / 4; j += 4) *reinterpret_cast<floatx4*>(dst + j) = (floatx4){o[j], o[j + 1], o[j + 2], o[j + 3]};
      if (g == 0) {
        p.ws_ml[2 * w] = m * p.c;
        p.ws_ml[2 * w + 1] = l;
      }
    } else {
      const float inv = l > 0.f ? 1.f / l : 0.f;
      uint16_t* dst = p.o + b * p.so[0] + h * p.so[1] + i * p.so[2] + g * (D / 4);
#pragma unroll
      for (int j = 0; j < D / 4; j += 4)
        *reinterpret_cast<u32x2*>(dst + j) = (u32x2){E::pack2(o[j] * inv, o[j + 1] * inv), E::pack2(o[j + 2] * inv, o[j + 3] * inv)};
      if (g == 0 && p.lse != nullptr)
        p.lse[b * p.sl[0] + h * p.sl[1] + i * p.sl[2]] =
            l > 0.f ? (m * p.c + __builtin_amdgcn_logf(l) - Fp4<Tag>::kPBias) * 0.6931471805599453f : FA_NEG_INF;
    }
  }

  __device__ static void run(const Kv4AttendParams& p, float* smem) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    // splits innermost: a sequence's neighbours run together; row blocks of one split share its tiles in L2
    const int rb = id % p.row_blocks;
    id /= p.row_blocks;
    const int split = id % p.splits;
    id /= p.splits;
    const int hk = id % p.Hkv, b = id / p.Hkv;
    const int rows = p.M * p.group;
    const int row0 = (SHARED ? rb : rb * WAVES + wave) * 16 * R;
    const int keys = visible_keys(p.start, p.count, b, p.M, p.capacity);
    const int per = tiles_per_split(keys, p.splits, p.min_tiles);
    if (split > 0 && split * per >= (keys + 31) / 32) return;  // behind the last key: the merge does not read it
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
    int least = wave_see;  // keys that every row of the wave sees
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
    }
    const int tiles = (wave_see + 31) / 32;
    int t0 = split * per, t1 = t0 + per < tiles ? t0 + per : tiles;
    const uint8_t* kc = p.k_codes + b * p.code_stride[0] + hk * p.code_stride[1];
    const uint8_t* vc = p.v_codes + b * p.code_stride[0] + hk * p.code_stride[1];
    const uint8_t* ks = p.k_scales + b * p.scale_stride[0] + hk * p.scale_stride[1];
    const uint8_t* vs = p.v_scales + b * p.scale_stride[0] + hk * p.scale_stride[1];
    const int stride = SHARED ? WAVES : 1;
    if (SHARED) t0 += wave;
    Tile now, next;
    if (t0 < t1) load(now, kc, ks, vc, vs, t0 * 32, lane);
    for (int t = t0; t < t1; t += stride) {
      if (t + stride < t1) load(next, kc, ks, vc, vs, (t + stride) * 32, lane);
      if (t * 32 + 32 <= least) step<false>(s, qf, now, t * 32, see, keys, p.c, lane);
      else step<true>(s, qf, now, t * 32, see, keys, p.c, lane);
      now = next;
    }
    if constexpr (SHARED) {
      // the waves' sums meet in LDS; wave w finishes rows 4 w .. 4 w + 3 of each 16
      constexpr int ROW = D + 4;
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        float l = s.l[rt];
        l = xquad_sum(l);
        float* dst = smem + (wave * 16 + c16) * ROW;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int d = 0; d < CPL; ++d) dst[(4 * g + r) * CPL + d] = s.o[d][rt][r];
        if (g == 0) {
          dst[D] = s.m[rt];
          dst[D + 1] = l;
        }
        __syncthreads();
        const int row = 4 * wave + (c16 & 3);
        if (c16 < 4) {
          float m = FA_NEG_INF;
#pragma unroll
          for (int w = 0; w < WAVES; ++w) m = fmaxf(m, smem[(w * 16 + row) * ROW + D]);
          float sum = 0.f, o[D / 4];
#pragma unroll
          for (int j = 0; j < D / 4; ++j) o[j] = 0.f;
#pragma unroll
          for (int w = 0; w < WAVES; ++w) {
            const float* src = smem + (w * 16 + row) * ROW;
            const float mw = src[D];
            const float f = mw == FA_NEG_INF && m == FA_NEG_INF ? 1.f : fast_exp2((mw - m) * p.c);
            sum += f * src[D + 1];
#pragma unroll
            for (int j = 0; j < D / 4; ++j) o[j] = fmaf(f, src[g * (D / 4) + j], o[j]);
          }
          const int r = row0 + 16 * rt + row;
          if (r < rows) store_row(p, b, hk, split, r, o, m, sum, g);
        }
        __syncthreads();
      }
    } else {
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        const float l = xquad_sum(s.l[rt]);
        float o[D / 4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int d = 0; d < CPL; ++d) o[r * CPL + d] = s.o[d][rt][r];
        const int r = row0 + 16 * rt + c16;
        if (r < rows) store_row(p, b, hk, split, r, o, s.m[rt], l, g);
      }
    }
  }
};

template <typename Tag, int D, int R, bool SHARED>
__global__ __launch_bounds__(256) void kv4_attend_kernel(Kv4AttendParams p) {
  __shared__ float smem[SHARED ? 4 * 16 * (D + 4) : 1];
  Kv4Attend<Tag, D, R, SHARED>::run(p, smem);
}

// Joins the splits of a row (one wave): weights exp2(m_s - m) of the unnormalised partial sums.
template <typename Tag, int D>
__global__ __launch_bounds__(256) void kv4_merge_kernel(Kv4AttendParams p) {
  constexpr int PL = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t rows = (int64_t)p.B * p.H * p.M;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int i = (int)(row % p.M);
  const int64_t bh = row / p.M;
  const int h = (int)(bh % p.H), b = (int)(bh / p.H);
  const int keys = visible_keys(p.start, p.count, b, p.M, p.capacity);
  const int tiles = (keys + 31) / 32;
  const int per = tiles_per_split(keys, p.splits, p.min_tiles);
  const int used = (tiles + per - 1) / per;
  float m = FA_NEG_INF;
  for (int s = lane; s < used; s += 64) m = fmaxf(m, p.ws_ml[2 * (s * rows + row)]);
#pragma unroll
  for (int k = 32; k >= 1; k /= 2) m = fmaxf(m, __shfl_xor(m, k, 64));
  float sum = 0.f, o[PL];
#pragma unroll
  for (int j = 0; j < PL; ++j) o[j] = 0.f;
  for (int s = 0; s < used; ++s) {
    const float ms = p.ws_ml[2 * (s * rows + row)];
    const float f = ms == FA_NEG_INF && m == FA_NEG_INF ? 1.f : fast_exp2(ms - m);
    sum = fmaf(f, p.ws_ml[2 * (s * rows + row) + 1], sum);
    const float* src = p.ws_o + (s * rows + row) * D + lane * PL;
#pragma unroll
    for (int j = 0; j < PL; ++j) o[j] = fmaf(f, src[j], o[j]);
  }
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  uint16_t* dst = p.o + b * p.so[0] + h * p.so[1] + i * p.so[2] + lane * PL;
#pragma unroll
  for (int j = 0; j < PL; ++j) dst[j] = DT<Tag>::from_float(o[j] * inv);
  if (lane == 0 && p.lse != nullptr)
    p.lse[b * p.sl[0] + h * p.sl[1] + i * p.sl[2]] =
        sum > 0.f ? (m + __builtin_amdgcn_logf(sum) - Fp4<Tag>::kPBias) * 0.6931471805599453f : FA_NEG_INF;
}

#define KV4_ENTRY(TAG, DTYPE, D)                                                                                   \
  {DTYPE, D, (const void*)&kv4_append_kernel<TAG>, (const void*)&kv4_merge_kernel<TAG, D>,                         \
   {(const void*)&kv4_attend_kernel<TAG, D, 1, true>, (const void*)&kv4_attend_kernel<TAG, D, 2, true>,            \
    (const void*)&kv4_attend_kernel<TAG, D, (D == 256 ? 1 : 2), false>}, D == 256 ? 1 : 2}

static const Kv4KernelEntry kKv4Entries[] = {
    KV4_ENTRY(f16_t, FA_DTYPE_F16, 64),   KV4_ENTRY(f16_t, FA_DTYPE_F16, 128),   KV4_ENTRY(f16_t, FA_DTYPE_F16, 256),
    KV4_ENTRY(bf16_t, FA_DTYPE_BF16, 64), KV4_ENTRY(bf16_t, FA_DTYPE_BF16, 128), KV4_ENTRY(bf16_t, FA_DTYPE_BF16, 256),
};

const Kv4KernelEntry* kv4_registry(int* count) {
  *count = (int)(sizeof(kKv4Entries) / sizeof(kKv4Entries[0]));
  return kKv4Entries;
}

}  // namespace fa
